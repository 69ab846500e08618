// The int8 Linear forward for a token or a few (decoding): igemm.cuh's z and its bits, without the
// tensor cores. What bounds it is reading W once and, in most layers, the latency of starting: here a
// thread's first instructions are its loads of W, where a tile on the tensor cores first sets up
// barriers, tensor memory and a cluster, and ends with an exchange between CTAs.
//
// A block takes 8 channels. Each of its warps takes 512 bytes of the rows in every 512 * warps: a lane
// reads 16 bytes of all eight and of the tokens' rows, two such steps of W in flight, and multiplies
// with dp4a. Eight channels, since each read of a token's bytes serves them all (with two channels and
// eight steps 12288 channels x K 1024 took 7.1 us, so 4.8), two steps, since a row of 1024 is done then.
// A warp's sums are added with redux, the warps' in shared memory, exact in any order; the first warp
// stores, a lane for each token and channel. One token measured: 4096 x 4096 5.2 us (3.2 TB/s; an
// empty launch takes 2.1), 12288 x 12288 25.9 us (5.8 TB/s). Four tokens are bound by the dp4a: 35 us.
//
// Rows start on 16 bytes, so a 16-byte read that holds an element of the row stays inside the row's
// stride, or, in the last row, inside the aligned 16 bytes that hold its last element. What lies past K
// is multiplied by zeros: the tokens' bytes there are cleared.
#pragma once

#include "common.cuh"
#include "igemm.cuh"

namespace c3cu {
namespace igemv {

constexpr int kMaxTokens = 4;  // x kChannels = the 32 lanes of the storing warp
constexpr int kChannels = 8;
constexpr int kMaxSplit = 16;
constexpr int kAhead = 2;   // steps of W in flight: 16 loads of 16 bytes a thread
constexpr int kStep = 512;  // bytes of a row that a warp reads at a time

__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int c) {
  c = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), c);
  c = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), c);
  c = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), c);
  return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), c);
}

// The first `n` bytes of v; the others zero.
__device__ __forceinline__ uint4 keep_bytes(uint4 v, int n) {
  const auto part = [n](uint32_t w, int at) {
    const int k = n - at;
    return k >= 4 ? w : k <= 0 ? 0u : w & ((1u << (8 * k)) - 1u);
  };
  return make_uint4(part(v.x, 0), part(v.y, 4), part(v.z, 8), part(v.w, 12));
}

template <int T, bool F32, bool RELU>
__global__ void __launch_bounds__(32 * kMaxSplit)
    igemv_kernel(const int8_t* __restrict__ px, int64_t ldx, const int8_t* __restrict__ pw, int64_t ldw,
                 const igemm::Params p) {
  constexpr int C = kChannels;
  __shared__ int s_sum[kMaxSplit][T][kChannels];
  const int lane = static_cast<int>(threadIdx.x & 31u);
  const int warp = static_cast<int>(threadIdx.x >> 5);
  const int split = static_cast<int>(blockDim.x >> 5);
  const int n0 = static_cast<int>(blockIdx.x) * kChannels;
  pdl_wait();
  pdl_launch_dependents();

  int sum[C][T];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int t = 0; t < T; ++t) sum[c][t] = 0;
  if (n0 < p.N) {
    const int8_t* w[C];
    const int8_t* x[T];
#pragma unroll
    for (int c = 0; c < C; ++c)  // past the last channel its row again: those sums are not stored
      w[c] = pw + static_cast<int64_t>(min(n0 + c, p.N - 1)) * ldw;
#pragma unroll
    for (int t = 0; t < T; ++t) x[t] = px + static_cast<int64_t>(min(t, p.M - 1)) * ldx;
    const int stride = kStep * split;
    for (int k0 = warp * kStep + lane * 16; k0 < p.K; k0 += kAhead * stride) {
      uint4 v[kAhead][C];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * stride;
        if (k < p.K) {
#pragma unroll
          for (int c = 0; c < C; ++c) v[i][c] = __ldg(reinterpret_cast<const uint4*>(w[c] + k));
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * stride;
        if (k >= p.K) break;
#pragma unroll
        for (int t = 0; t < T; ++t) {
          uint4 u = __ldg(reinterpret_cast<const uint4*>(x[t] + k));
          if (k + 16 > p.K) u = keep_bytes(u, p.K - k);
#pragma unroll
          for (int c = 0; c < C; ++c) sum[c][t] = dot16(v[i][c], u, sum[c][t]);
        }
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int t = 0; t < T; ++t) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int s = __reduce_add_sync(0xffffffffu, sum[c][t]);
      if (lane == 0) s_sum[warp][t][c] = s;
    }
  }
  __syncthreads();
  if (warp != 0) return;
  const int t = lane / C, c = lane % C;
  const bool in = t < T && t < p.M && n0 + c < p.N;
  float z = 0.f;
  if (in) {
    int acc = 0;
    for (int s = 0; s < split; ++s) acc += s_sum[s][t][c];
    z = __fmul_rn(__int2float_rn(acc), __fmul_rn(__ldg(p.xs + t), __ldg(p.ws + n0 + c)));
    if (p.bias) z = __fadd_rn(z, __ldg(p.bias + n0 + c));
  }
  if constexpr (RELU) {
    if (p.mask) {  // a byte of the token's mask; the blocks past N clear the rest of the last word
      const uint32_t bits = __ballot_sync(0xffffffffu, in && z > 0.f);
      if (c == 0 && t < T && t < p.M)
        reinterpret_cast<uint8_t*>(p.mask + static_cast<int64_t>(t) * p.ldm)[blockIdx.x] =
            static_cast<uint8_t>(bits >> lane);
    }
    z = igemm::relu_keep_nan(z);
  }
  if (!in) return;
  const int64_t at = static_cast<int64_t>(t) * p.ldo + n0 + c;
  if constexpr (F32) static_cast<float*>(p.out)[at] = z;
  else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(z);
}

}  // namespace igemv
}  // namespace c3cu
