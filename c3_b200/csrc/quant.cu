// Row-wise kernels of the 8-bit activation path (include/c3cu.h):
//   * c3cu_quantize_rows  — q = round(127 x / A), scale = A / 127, A = max |x| of the row
//   * c3cu_rms_norm_int8  — h = x + residual, rstd = 1 / sqrt(mean h^2 + eps), and
//                           y = h * rstd * weight in the same int8 form
//   * c3cu_rms_norm_bwd   — the norm's gradients dx (+ the gradient reaching h directly) and
//                           dweight; the rounding to int8 counts as the identity
// The reference has no counterpart (its kernels are fp32 throughout).
//
// The int8 numbers do not depend on rstd: with a = fl32(h * w) and A = max |a| the row's q is
// round(127 a / A), so one reduction over the row yields both the sum of squares and A, and a
// row is read once. q is the integer nearest to the real quotient, ties to even, whatever the
// launch shape: an element whose fp32 quotient lies too near to a half-integer to be decided is
// divided again in fp64, which decides every case (a and A have 24-bit significands, so a
// quotient that is not a tie is at least 2^-32 of its size away from one).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "host_util.h"

namespace c3cu {
namespace quant {

// ---------------------------------------------------------------- element access
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float round(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
};

// V consecutive elements as fp32; V is 1 or one 16-byte vector. Inputs are streamed: each is read once.
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = static_cast<float>(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 r = __ldcs(reinterpret_cast<const float4*>(p));
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  } else {
    const uint4 r = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (sizeof(T) == 4) *p = v[0];
    else *p = __float2bfloat16_rn(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// fp32 weights stay in L1 / L2: every row reads them.
template <int V>
__device__ __forceinline__ void load_weight(const float* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = __ldg(p);
  } else {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float4 r = __ldg(reinterpret_cast<const float4*>(p) + j);
      v[4 * j] = r.x; v[4 * j + 1] = r.y; v[4 * j + 2] = r.z; v[4 * j + 3] = r.w;
    }
  }
}

// ---------------------------------------------------------------- rounding to int8
__device__ __noinline__ int quantize_exact(float a, float big) {
  return static_cast<int>(rint(127.0 * static_cast<double>(a) / static_cast<double>(big)));
}

struct RowScale {
  float big;   // A
  float inv;   // 127 / A
  float safe;  // largest |t - round(t)| at which t = a * inv rounds like the real quotient
  bool finite;
};

// `bits` is the largest |a| as its bit pattern (which orders like the number, with infinities and
// NaN on top).
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale r;
  r.big = __uint_as_float(bits);
  r.finite = bits < 0x7f800000u;
  r.inv = r.finite && bits != 0u ? __fdiv_rn(127.f, r.big) : 0.f;
  // t carries two roundings, an error of at most 127 * 2^-23 = 1.6e-5. Below 1e-35 the reciprocal
  // could overflow: every element takes the fp64 division.
  r.safe = (bits == 0u || r.big > 1e-35f) ? 0.5f - 6.1e-5f : -1.f;
  return r;
}

template <int V>
__device__ __forceinline__ void store_q(int8_t* q, const float* a, const RowScale& r) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it leaves round(t) in the low bits
  uint32_t n[V];
  float off[V];
  float worst = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float t = __fmul_rn(a[j], r.inv);
    const float m = __fadd_rn(t, kMagic);
    n[j] = __float_as_uint(m);
    off[j] = fabsf(__fsub_rn(t, __fsub_rn(m, kMagic)));
    worst = fmaxf(worst, off[j]);
  }
  if (worst > r.safe) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!(off[j] <= r.safe)) n[j] = static_cast<uint32_t>(quantize_exact(a[j], r.big));
  }
  if (!r.finite) {
#pragma unroll
    for (int j = 0; j < V; ++j) n[j] = 0u;
  }
  if constexpr (V == 1) {
    *q = static_cast<int8_t>(n[0]);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j)
      w[j] = __byte_perm(__byte_perm(n[4 * j], n[4 * j + 1], 0x0040),
                         __byte_perm(n[4 * j + 2], n[4 * j + 3], 0x0040), 0x5410);
    if constexpr (V == 4) *reinterpret_cast<uint32_t*>(q) = w[0];
    else *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
  }
}

// ---------------------------------------------------------------- reductions over a row
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum and bit-pattern maximum over the block (WARP: over the warp), the same on every thread.
template <bool WARP>
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& top) {
  sum = warp_sum(sum);
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (!WARP) {
    __shared__ float s_sum[32];
    __shared__ uint32_t s_top[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
      s_sum[warp] = sum;
      s_top[warp] = top;
    }
    __syncthreads();
    sum = warp_sum(lane < warps ? s_sum[lane] : 0.f);
    top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[lane] : 0u);
  }
}

__device__ __forceinline__ float rstd_of(float sum_squares, int K, float eps) {
  return __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum_squares, static_cast<float>(K)), eps)));
}

// ---------------------------------------------------------------- quantise / norm forward
struct FwdArgs {
  const void* x;
  const void* res;      // RES: added to x
  const float* weight;  // NORM
  void* h;              // RES: the rounded sum
  int8_t* q;
  float* scale;
  float* rstd;          // NORM
  int64_t ldx, ldr, ldh, ldq;
  int M, K;
  float eps;
};

__device__ __forceinline__ void row_outputs(const FwdArgs& p, int64_t row, float sum, const RowScale& r, bool norm) {
  float s = r.big;
  if (norm) {
    const float rs = rstd_of(sum, p.K, p.eps);
    p.rstd[row] = rs;
    s = __fmul_rn(s, rs);
  }
  p.scale[row] = r.finite ? __fdiv_rn(s, 127.f) : __int_as_float(0x7fc00000);
}

// One row per block (or per warp), held in registers between the reduction and the rounding:
// N vectors of V elements per thread.
template <typename T, bool NORM, bool RES, int V, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) rows_kernel(const FwdArgs p) {
  const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)
                           : static_cast<int64_t>(blockIdx.x);
  if (WARP && row >= p.M) return;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int G = WARP ? 32 : blockDim.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float a[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * G) * V;
    if (c < p.K) load<T, V>(x + c, a[i]);
    else
#pragma unroll
      for (int j = 0; j < V; ++j) a[i][j] = 0.f;
  }
  if constexpr (RES) {
    const T* r = static_cast<const T*>(p.res) + row * p.ldr;
    T* h = static_cast<T*>(p.h) + row * p.ldh;
    float b[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * G) * V;
      if (c < p.K) load<T, V>(r + c, b[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * G) * V;
      if (c < p.K) {
#pragma unroll
        for (int j = 0; j < V; ++j) a[i][j] = Elem<T>::round(__fadd_rn(a[i][j], b[i][j]));
        store<T, V>(h + c, a[i]);
      }
    }
  }
  float sum = 0.f;
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (NORM) {
      const int c = (t + i * G) * V;
      float w[V];
      if (c < p.K) load_weight<V>(p.weight + c, w);
      else
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        sum = fmaf(a[i][j], a[i][j], sum);
        a[i][j] = __fmul_rn(a[i][j], w[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(a[i][j]) & 0x7fffffffu);
  }
  row_reduce<WARP>(sum, top);
  const RowScale r = row_scale(top);
  int8_t* q = p.q + row * p.ldq;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * G) * V;
    if (c < p.K) store_q<V>(q + c, a[i], r);
  }
  if (t == 0) row_outputs(p, row, sum, r, NORM);
}

// Rows too long for the registers of a block: two passes over the row. The second reads x again
// (or h, which each thread wrote itself).
template <typename T, bool NORM, bool RES, int V>
__global__ void __launch_bounds__(1024) long_rows_kernel(const FwdArgs p) {
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* r = RES ? static_cast<const T*>(p.res) + row * p.ldr : nullptr;
  T* h = RES ? static_cast<T*>(p.h) + row * p.ldh : nullptr;
  float sum = 0.f;
  uint32_t top = 0u;
  for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < p.K; c += static_cast<int64_t>(blockDim.x) * V) {
    float a[V];
    load<T, V>(x + c, a);
    if constexpr (RES) {
      float b[V];
      load<T, V>(r + c, b);
#pragma unroll
      for (int j = 0; j < V; ++j) a[j] = Elem<T>::round(__fadd_rn(a[j], b[j]));
      store<T, V>(h + c, a);
    }
    if constexpr (NORM) {
      float w[V];
      load_weight<V>(p.weight + c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        sum = fmaf(a[j], a[j], sum);
        a[j] = __fmul_rn(a[j], w[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(a[j]) & 0x7fffffffu);
  }
  row_reduce<false>(sum, top);
  const RowScale rs = row_scale(top);
  int8_t* q = p.q + row * p.ldq;
  const T* again = RES ? h : x;
  for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < p.K; c += static_cast<int64_t>(blockDim.x) * V) {
    float a[V];
    load<T, V>(again + c, a);
    if constexpr (NORM) {
      float w[V];
      load_weight<V>(p.weight + c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) a[j] = __fmul_rn(a[j], w[j]);
    }
    store_q<V>(q + c, a, rs);
  }
  if (threadIdx.x == 0) row_outputs(p, row, sum, rs, NORM);
}

// ---------------------------------------------------------------- norm backward
struct BwdArgs {
  const void* dy;
  const void* h;
  const void* dh;  // may be null
  const float* weight;
  const float* rstd;
  void* dx;
  float* dweight;
  float* partial;  // [grid][K], unless one block does all rows
  int64_t ldy, ldhh, lddh, lddx;
  int M, K;
};

// g = w dy, xhat = h rstd: dx = rstd (g - xhat mean(g xhat)) + dh, dweight = sum_rows dy xhat.
// A block walks over rows (grid-strided); a thread owns the same N x V columns in each, so
// dweight's share of the block stays in registers until the end.
template <typename T, int V, int N>
__global__ void __launch_bounds__(768) norm_bwd_kernel(const BwdArgs p) {
  const int t = threadIdx.x, G = blockDim.x;
  float w[N][V], acc[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * G) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) w[i][j] = acc[i][j] = 0.f;
    if (c < p.K) load_weight<V>(p.weight + c, w[i]);
  }
  const float inv_k = __fdiv_rn(1.f, static_cast<float>(p.K));
  __shared__ float s_sum[2][32];
  int flip = 0;
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x, flip ^= 1) {
    const T* dy = static_cast<const T*>(p.dy) + row * p.ldy;
    const T* h = static_cast<const T*>(p.h) + row * p.ldhh;
    float g[N][V], xh[N][V], d[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * G) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) g[i][j] = xh[i][j] = d[i][j] = 0.f;
      if (c < p.K) {
        load<T, V>(dy + c, g[i]);
        load<T, V>(h + c, xh[i]);
        if (p.dh) load<T, V>(static_cast<const T*>(p.dh) + row * p.lddh + c, d[i]);
      }
    }
    const float rs = __ldg(p.rstd + row);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[i][j] *= rs;
        acc[i][j] = fmaf(g[i][j], xh[i][j], acc[i][j]);
        g[i][j] *= w[i][j];
        dot = fmaf(g[i][j], xh[i][j], dot);
      }
    dot = warp_sum(dot);
    // two buffers: a warp may be one row ahead of the warps still reading the last row's sums
    if ((t & 31) == 0) s_sum[flip][t >> 5] = dot;
    __syncthreads();
    dot = warp_sum((t & 31) < (G >> 5) ? s_sum[flip][t & 31] : 0.f) * inv_k;
    T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * G) * V;
      if (c < p.K) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = fmaf(rs, fmaf(-xh[i][j], dot, g[i][j]), d[i][j]);
        store<T, V>(dx + c, d[i]);
      }
    }
  }
  float* out = gridDim.x == 1 ? p.dweight : p.partial + static_cast<int64_t>(blockIdx.x) * p.K;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * G) * V;
    if (c < p.K) {
#pragma unroll
      for (int j = 0; j < V; ++j) out[c + j] = acc[i][j];
    }
  }
}

// Long rows: the row's dot product first, then dx and dweight by strips of 32 columns.
template <typename T>
__global__ void __launch_bounds__(1024) norm_bwd_dot_kernel(const BwdArgs p, float* __restrict__ dots) {
  const int64_t row = blockIdx.x;
  const T* dy = static_cast<const T*>(p.dy) + row * p.ldy;
  const T* h = static_cast<const T*>(p.h) + row * p.ldhh;
  const float rs = __ldg(p.rstd + row);
  float dot = 0.f;
  for (int64_t c = threadIdx.x; c < p.K; c += blockDim.x)
    dot = fmaf(static_cast<float>(dy[c]) * __ldg(p.weight + c), static_cast<float>(h[c]) * rs, dot);
  uint32_t unused = 0u;
  row_reduce<false>(dot, unused);
  if (threadIdx.x == 0) dots[row] = dot / static_cast<float>(p.K);
}

template <typename T>
__global__ void __launch_bounds__(256) norm_bwd_strip_kernel(const BwdArgs p, const float* __restrict__ dots,
                                                             int rows_per_block) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int warp = threadIdx.x >> 5;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t r1 = min(r0 + rows_per_block, static_cast<int64_t>(p.M));
  float acc = 0.f;
  if (c < p.K) {
    const float w = __ldg(p.weight + c);
    for (int64_t row = r0 + warp; row < r1; row += 8) {
      const float rs = __ldg(p.rstd + row);
      const float dy = static_cast<float>(static_cast<const T*>(p.dy)[row * p.ldy + c]);
      const float xh = static_cast<float>(static_cast<const T*>(p.h)[row * p.ldhh + c]) * rs;
      const float d = p.dh ? static_cast<float>(static_cast<const T*>(p.dh)[row * p.lddh + c]) : 0.f;
      acc = fmaf(dy, xh, acc);
      const float v[1] = {fmaf(rs, fmaf(-xh, dots[row], dy * w), d)};
      store<T, 1>(static_cast<T*>(p.dx) + row * p.lddx + c, v);
    }
  }
  __shared__ float part[8][32];
  part[warp][threadIdx.x & 31] = acc;
  __syncthreads();
  if (warp == 0 && c < p.K) {
#pragma unroll
    for (int i = 1; i < 8; ++i) acc += part[i][threadIdx.x];
    (gridDim.y == 1 ? p.dweight : p.partial + static_cast<int64_t>(blockIdx.y) * p.K)[c] = acc;
  }
}

// dweight = sum of the blocks' shares, in a fixed order.
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* __restrict__ partial, float* __restrict__ out,
                                                           int rows, int K) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int warp = threadIdx.x >> 5;
  float acc = 0.f;
  if (c < K) {
#pragma unroll 8
    for (int r = warp; r < rows; r += 8) acc += __ldcs(partial + static_cast<int64_t>(r) * K + c);
  }
  __shared__ float part[8][32];
  part[warp][threadIdx.x & 31] = acc;
  __syncthreads();
  if (warp == 0 && c < K) {
#pragma unroll
    for (int i = 1; i < 8; ++i) acc += part[i][threadIdx.x];
    out[c] = acc;
  }
}

// ---------------------------------------------------------------- launch rules
inline bool rows_aligned(const void* p, int64_t ld, int64_t M, int esize, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (M <= 1 || ld * esize % bytes == 0);
}

template <typename T, bool NORM, bool RES, int V, int N>
cudaError_t launch_rows_n(const FwdArgs& p, cudaStream_t st) {
  const int need = (p.K + V * N - 1) / (V * N);  // threads for a row
  if (need <= 32) {
    const int per = 4;
    rows_kernel<T, NORM, RES, V, N, true><<<(p.M + per - 1) / per, 32 * per, 0, st>>>(p);
  } else {
    rows_kernel<T, NORM, RES, V, N, false><<<p.M, (need + 31) / 32 * 32, 0, st>>>(p);
  }
  return cudaGetLastError();
}

// 16 elements per thread keep enough loads in flight; a row over 16 * 1024 elements takes two passes.
template <typename T, bool NORM, bool RES>
cudaError_t launch_rows(const FwdArgs& p, bool vec, cudaStream_t st) {
  constexpr int V = Elem<T>::kVec;
  if (vec) {
    if (p.K <= 16 * 1024) return launch_rows_n<T, NORM, RES, V, 16 / V>(p, st);
    long_rows_kernel<T, NORM, RES, V><<<p.M, 1024, 0, st>>>(p);
  } else {
    if (p.K <= 16 * 1024) return launch_rows_n<T, NORM, RES, 1, 16>(p, st);
    long_rows_kernel<T, NORM, RES, 1><<<p.M, 1024, 0, st>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
int fwd(const FwdArgs& p, bool norm, cudaStream_t st, const char* what) {
  constexpr int V = Elem<T>::kVec;
  const int e = static_cast<int>(sizeof(T));
  bool vec = p.K % V == 0 && rows_aligned(p.x, p.ldx, p.M, e, 16) && rows_aligned(p.q, p.ldq, p.M, 1, V);
  if (norm) vec = vec && aligned16(p.weight);
  if (p.res) vec = vec && rows_aligned(p.res, p.ldr, p.M, e, 16) && rows_aligned(p.h, p.ldh, p.M, e, 16);
  cudaError_t err = !norm ? launch_rows<T, false, false>(p, vec, st)
                   : p.res ? launch_rows<T, true, true>(p, vec, st) : launch_rows<T, true, false>(p, vec, st);
  return cuda_status(err, what);
}

constexpr int kBwdCols = 16;              // columns a thread owns
constexpr int kBwdMaxK = 768 * kBwdCols;  // beyond: strips

// Rows of a strip block: 256, or what keeps the grid's y dimension inside its limit.
int strip_rows(int64_t M) { return M <= 256 * int64_t{65535} ? 256 : static_cast<int>((M + 65534) / 65535); }

int bwd_grid(int64_t M, int64_t K) {
  const int threads = static_cast<int>((K + kBwdCols * 32 - 1) / (kBwdCols * 32)) * 32;
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const int per_sm = threads >= 768 ? 1 : (threads > 256 ? 2 : (threads > 128 ? 3 : 6));
  const int64_t most = static_cast<int64_t>(sms) * per_sm;
  return static_cast<int>(M < most ? M : most);
}

size_t bwd_partial_rows(int64_t M, int64_t K) {
  return K <= kBwdMaxK ? static_cast<size_t>(bwd_grid(M, K)) : static_cast<size_t>((M + strip_rows(M) - 1) / strip_rows(M));
}

template <typename T>
int bwd(BwdArgs p, bool vec, float* ws, cudaStream_t st) {
  constexpr int V = Elem<T>::kVec;
  const int rows = static_cast<int>(bwd_partial_rows(p.M, p.K));
  if (p.K <= kBwdMaxK) {
    const int threads = (p.K + kBwdCols * 32 - 1) / (kBwdCols * 32) * 32;
    p.partial = ws;
    if (vec) norm_bwd_kernel<T, V, kBwdCols / V><<<rows, threads, 0, st>>>(p);
    else norm_bwd_kernel<T, 1, kBwdCols><<<rows, threads, 0, st>>>(p);
  } else {
    float* dots = ws;
    p.partial = ws + p.M;
    norm_bwd_dot_kernel<T><<<p.M, 1024, 0, st>>>(p, dots);
    norm_bwd_strip_kernel<T><<<dim3((p.K + 31) / 32, rows), 256, 0, st>>>(p, dots, strip_rows(p.M));
  }
  int rc = cuda_status(cudaGetLastError(), "rms_norm_bwd: launch");
  if (rc != C3CU_OK || rows <= 1) return rc;
  sum_partials_kernel<<<(p.K + 31) / 32, 256, 0, st>>>(p.partial, p.dweight, rows, p.K);
  return cuda_status(cudaGetLastError(), "rms_norm_bwd: launch");
}

int check_sizes(const char* what, int64_t M, int64_t K, int dtype) {
  if (dtype != C3CU_DTYPE_F32 && dtype != C3CU_DTYPE_BF16) {
    set_error("%s: dtype %d is neither f32 nor bf16", what, dtype);
    return C3CU_ERR_INVALID;
  }
  if (M < 0 || K < 1 || M > INT32_MAX || K > INT32_MAX) {
    set_error("%s: sizes out of range (M %lld, K %lld; K >= 1)", what, (long long)M, (long long)K);
    return C3CU_ERR_INVALID;
  }
  return C3CU_OK;
}

int check_ld(const char* what, const char* name, const void* p, int64_t ld, int64_t M, int64_t K, int align) {
  if (!p) {
    set_error("%s: %s is null", what, name);
    return C3CU_ERR_INVALID;
  }
  if (M > 1 && ld < K) {
    set_error("%s: row stride %lld of %s is smaller than K %lld", what, (long long)ld, name, (long long)K);
    return C3CU_ERR_INVALID;
  }
  if (reinterpret_cast<uintptr_t>(p) % align != 0) {
    set_error("%s: %s is not aligned to its type", what, name);
    return C3CU_ERR_ALIGN;
  }
  return C3CU_OK;
}

}  // namespace quant
}  // namespace c3cu

#define C3CU_TRY(expr)               \
  do {                               \
    const int rc_ = (expr);          \
    if (rc_ != C3CU_OK) return rc_;  \
  } while (0)

extern "C" int c3cu_quantize_rows(const void* X, int64_t ldx, int dtype, int8_t* Q, int64_t ldq, float* scale,
                                  int64_t M, int64_t K, c3cu_stream_t stream) {
  using namespace c3cu;
  const char* what = "quantize_rows";
  C3CU_TRY(require_sm100());
  C3CU_TRY(quant::check_sizes(what, M, K, dtype));
  if (M == 0) return C3CU_OK;
  C3CU_TRY(quant::check_ld(what, "X", X, ldx, M, K, dtype == C3CU_DTYPE_F32 ? 4 : 2));
  C3CU_TRY(quant::check_ld(what, "Q", Q, ldq, M, K, 1));
  C3CU_TRY(quant::check_ld(what, "scale", scale, K, M, K, 4));
  quant::FwdArgs p{};
  p.x = X; p.q = Q; p.scale = scale;
  p.ldx = ldx; p.ldq = ldq;
  p.M = static_cast<int>(M); p.K = static_cast<int>(K);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == C3CU_DTYPE_F32 ? quant::fwd<float>(p, false, st, "quantize_rows: launch")
                                 : quant::fwd<__nv_bfloat16>(p, false, st, "quantize_rows: launch");
}

extern "C" int c3cu_rms_norm_int8(const void* X, int64_t ldx, const void* R, int64_t ldr, int dtype,
                                  const float* weight, float eps, void* H, int64_t ldh, int8_t* Q, int64_t ldq,
                                  float* scale, float* rstd, int64_t M, int64_t K, c3cu_stream_t stream) {
  using namespace c3cu;
  const char* what = "rms_norm_int8";
  C3CU_TRY(require_sm100());
  C3CU_TRY(quant::check_sizes(what, M, K, dtype));
  if (!(eps >= 0.f)) {
    set_error("%s: eps %g is negative or NaN", what, eps);
    return C3CU_ERR_INVALID;
  }
  if (M == 0) return C3CU_OK;
  const int e = dtype == C3CU_DTYPE_F32 ? 4 : 2;
  C3CU_TRY(quant::check_ld(what, "X", X, ldx, M, K, e));
  if ((R != nullptr) != (H != nullptr)) {
    set_error("%s: a residual and the sum's output come together (without a residual h is X itself)", what);
    return C3CU_ERR_INVALID;
  }
  if (R) {
    C3CU_TRY(quant::check_ld(what, "R", R, ldr, M, K, e));
    C3CU_TRY(quant::check_ld(what, "H", H, ldh, M, K, e));
  }
  C3CU_TRY(quant::check_ld(what, "Q", Q, ldq, M, K, 1));
  C3CU_TRY(quant::check_ld(what, "weight", weight, K, M, K, 4));
  C3CU_TRY(quant::check_ld(what, "scale", scale, K, M, K, 4));
  C3CU_TRY(quant::check_ld(what, "rstd", rstd, K, M, K, 4));
  quant::FwdArgs p{};
  p.x = X; p.res = R; p.weight = weight; p.h = H; p.q = Q; p.scale = scale; p.rstd = rstd;
  p.ldx = ldx; p.ldr = ldr; p.ldh = ldh; p.ldq = ldq;
  p.M = static_cast<int>(M); p.K = static_cast<int>(K);
  p.eps = eps;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == C3CU_DTYPE_F32 ? quant::fwd<float>(p, true, st, "rms_norm_int8: launch")
                                 : quant::fwd<__nv_bfloat16>(p, true, st, "rms_norm_int8: launch");
}

extern "C" size_t c3cu_rms_norm_bwd_workspace(int64_t M, int64_t K) {
  using namespace c3cu;
  if (M < 1 || K < 1) return 0;
  const size_t rows = quant::bwd_partial_rows(M, K);
  const size_t dots = K <= quant::kBwdMaxK ? 0 : static_cast<size_t>(M);
  return (dots + (rows > 1 ? rows * static_cast<size_t>(K) : 0)) * sizeof(float);
}

extern "C" int c3cu_rms_norm_bwd(const void* dY, int64_t ldy, const void* H, int64_t ldh, const void* dH, int64_t lddh,
                                 int dtype, const float* weight, const float* rstd, void* dX, int64_t lddx,
                                 float* dweight, int64_t M, int64_t K, void* workspace, size_t workspace_bytes,
                                 c3cu_stream_t stream) {
  using namespace c3cu;
  const char* what = "rms_norm_bwd";
  C3CU_TRY(require_sm100());
  C3CU_TRY(quant::check_sizes(what, M, K, dtype));
  const int e = dtype == C3CU_DTYPE_F32 ? 4 : 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  C3CU_TRY(quant::check_ld(what, "dweight", dweight, K, M, K, 4));
  if (M == 0)  // the sum over no rows
    return cuda_status(cudaMemsetAsync(dweight, 0, static_cast<size_t>(K) * sizeof(float), st), what);
  C3CU_TRY(quant::check_ld(what, "dY", dY, ldy, M, K, e));
  C3CU_TRY(quant::check_ld(what, "H", H, ldh, M, K, e));
  if (dH) C3CU_TRY(quant::check_ld(what, "dH", dH, lddh, M, K, e));
  C3CU_TRY(quant::check_ld(what, "weight", weight, K, M, K, 4));
  C3CU_TRY(quant::check_ld(what, "rstd", rstd, K, M, K, 4));
  C3CU_TRY(quant::check_ld(what, "dX", dX, lddx, M, K, e));
  const size_t need = c3cu_rms_norm_bwd_workspace(M, K);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    set_error("%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : size_t{0}, need);
    return C3CU_ERR_WORKSPACE;
  }
  if (need > 0) C3CU_TRY(quant::check_ld(what, "workspace", workspace, K, M, K, 4));
  quant::BwdArgs p{};
  p.dy = dY; p.h = H; p.dh = dH; p.weight = weight; p.rstd = rstd; p.dx = dX; p.dweight = dweight;
  p.ldy = ldy; p.ldhh = ldh; p.lddh = lddh; p.lddx = lddx;
  p.M = static_cast<int>(M); p.K = static_cast<int>(K);
  const int V = dtype == C3CU_DTYPE_F32 ? 4 : 8;
  const bool vec = K % V == 0 && aligned16(weight) && quant::rows_aligned(dY, ldy, M, e, 16) &&
                   quant::rows_aligned(H, ldh, M, e, 16) && (!dH || quant::rows_aligned(dH, lddh, M, e, 16)) &&
                   quant::rows_aligned(dX, lddx, M, e, 16);
  return dtype == C3CU_DTYPE_F32 ? quant::bwd<float>(p, vec, static_cast<float*>(workspace), st)
                                 : quant::bwd<__nv_bfloat16>(p, vec, static_cast<float*>(workspace), st);
}
