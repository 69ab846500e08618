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
#include <atomic>
#include <cstdlib>

#include "common.cuh"
#include "host_util.h"

C3CU_FAULT_ACCESSORS(quant)

namespace c3cu {
namespace quant {

constexpr int kRowElems = 16;  // elements of a row per thread, where a row is held in registers

// ---------------------------------------------------------------- packed fp32
// Two elements per instruction, each rounded like its scalar form.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}

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

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The largest magnitude of three, a NaN if there is one.
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ---------------------------------------------------------------- element access
// A thread works on runs of V elements, held as fp32 pairs. Where rows start on 16 bytes a run is
// one 16-byte vector (SG = 0). Elsewhere it is eight single elements SG apart, SG being the block's
// threads (a compile-time number, so that the eight addresses are one register and immediates): a
// warp still reads 32 neighbours at a time, and the arithmetic is the same packed one.
template <typename T, int SG>
struct Runs {
  static constexpr int V = SG ? 8 : 16 / static_cast<int>(sizeof(T));
  // the column of element j of run i, of thread t among G
  static __device__ __forceinline__ int col(int t, int i, int j, int G) {
    return SG ? t + (i * 8 + j) * SG : (t + i * G) * V + j;
  }
  // whether run i of the thread may have elements left of K
  static __device__ __forceinline__ bool any(int t, int i, int G, int K) {
    return SG ? i * 8 * SG < K : (t + i * G) * V < K;
  }
};

template <int V>
struct Run {
  float2 v[V / 2];
  __device__ __forceinline__ float operator[](int j) const { return j & 1 ? v[j / 2].y : v[j / 2].x; }
};

template <int V>
__device__ __forceinline__ void clear(Run<V>& x) {
#pragma unroll
  for (int j = 0; j < V / 2; ++j) x.v[j] = make_float2(0.f, 0.f);
}

__device__ __forceinline__ float2 unpack(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ void expand(const uint4& r, Run<16 / sizeof(T)>& x) {
  if constexpr (sizeof(T) == 4) {
    x.v[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    x.v[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  } else {
    x.v[0] = unpack(r.x);
    x.v[1] = unpack(r.y);
    x.v[2] = unpack(r.z);
    x.v[3] = unpack(r.w);
  }
}

// Run i of a row in global memory, zeros past K. Inputs are streamed: each is read once.
template <typename T, int SG>
__device__ __forceinline__ void load(const T* row, int t, int i, int G, int K, Run<Runs<T, SG>::V>& x) {
  using R = Runs<T, SG>;
  if constexpr (SG == 0) {
    const int c = R::col(t, i, 0, G);
    if (c < K) expand<T>(__ldcs(reinterpret_cast<const uint4*>(row + c)), x);
    else clear(x);
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = R::col(t, i, j, G);
      f[j] = c < K ? static_cast<float>(row[c]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = make_float2(f[2 * j], f[2 * j + 1]);
  }
}

// fp32 weights stay in L1 / L2: every row reads them.
template <typename T, int SG>
__device__ __forceinline__ void load_weight(const float* w, int t, int i, int G, int K, Run<Runs<T, SG>::V>& x) {
  using R = Runs<T, SG>;
  if constexpr (SG == 0) {
    const int c = R::col(t, i, 0, G);
    if (c < K) {
#pragma unroll
      for (int j = 0; j < R::V / 4; ++j) {
        const float4 r = __ldg(reinterpret_cast<const float4*>(w + c) + j);
        x.v[2 * j] = make_float2(r.x, r.y);
        x.v[2 * j + 1] = make_float2(r.z, r.w);
      }
    } else {
      clear(x);
    }
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = R::col(t, i, j, G);
      f[j] = c < K ? __ldg(w + c) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = make_float2(f[2 * j], f[2 * j + 1]);
  }
}

// Rounds run i to T, writes it, and keeps the rounded values.
template <typename T, int SG>
__device__ __forceinline__ void store(T* row, int t, int i, int G, int K, Run<Runs<T, SG>::V>& x) {
  using R = Runs<T, SG>;
  if constexpr (SG == 0) {
    const int c = R::col(t, i, 0, G);
    if (c >= K) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + c) = make_float4(x.v[0].x, x.v[0].y, x.v[1].x, x.v[1].y);
    } else {
      uint4 w;
      w.x = pack_bf16x2(x.v[0].x, x.v[0].y);
      w.y = pack_bf16x2(x.v[1].x, x.v[1].y);
      w.z = pack_bf16x2(x.v[2].x, x.v[2].y);
      w.w = pack_bf16x2(x.v[3].x, x.v[3].y);
      *reinterpret_cast<uint4*>(row + c) = w;
      expand<T>(w, x);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c0 = R::col(t, i, 2 * j, G), c1 = R::col(t, i, 2 * j + 1, G);
      if constexpr (sizeof(T) == 4) {
        if (c0 < K) row[c0] = x.v[j].x;
        if (c1 < K) row[c1] = x.v[j].y;
      } else {
        const uint32_t w = pack_bf16x2(x.v[j].x, x.v[j].y);
        if (c0 < K) row[c0] = __ushort_as_bfloat16(static_cast<unsigned short>(w));
        if (c1 < K) row[c1] = __ushort_as_bfloat16(static_cast<unsigned short>(w >> 16));
        x.v[j] = unpack(w);
      }
    }
  }
}

// Run i of a vector of fp32 sums.
template <typename T, int SG>
__device__ __forceinline__ void store_sums(float* out, int t, int i, int G, int K, const Run<Runs<T, SG>::V>& x) {
  using R = Runs<T, SG>;
#pragma unroll
  for (int j = 0; j < R::V; ++j) {
    const int c = R::col(t, i, j, G);
    if (c < K) out[c] = x[j];
  }
}

// ---------------------------------------------------------------- rounding to int8
__device__ __noinline__ uint32_t quantize_exact(float a, float big) {
  return static_cast<uint32_t>(static_cast<int>(rint(127.0 * static_cast<double>(a) / static_cast<double>(big))));
}

struct RowScale {
  float big;   // A
  float inv;   // 127 / A
  float safe;  // largest |a inv - round(a inv)| at which a inv rounds like the real quotient
  bool finite;
};

// `bits` is the largest |a| as its bit pattern (which orders like the number, with infinities and
// NaN on top).
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale r;
  r.big = __uint_as_float(bits);
  r.finite = bits < 0x7f800000u;
  float rcp;  // within 2^-23 of 1 / A
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rcp) : "f"(r.big));
  r.inv = r.finite && bits != 0u ? 127.f * rcp : 0.f;
  // a inv, multiplied without a rounding, is off by inv's: at most 127 * 1.5 * 2^-23 = 2.3e-5. Near
  // the ends of fp32's range the reciprocal may overflow or vanish: there every element takes the
  // fp64 division.
  r.safe = (bits == 0u || (r.big > 1e-35f && r.big < 1e37f)) ? 0.5f - 4e-5f : -1.f;
  return r;
}

template <typename T, int SG>
__device__ __forceinline__ void store_q(int8_t* row, int t, int i, int G, int K, const Run<Runs<T, SG>::V>& a,
                                        const RowScale& r) {
  using R = Runs<T, SG>;
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it leaves round(a inv) in the low bits
  uint32_t n[R::V];
  float off[R::V];
  float worst = 0.f;
#pragma unroll
  for (int j = 0; j < R::V / 2; ++j) {
    const float2 m = fma2(a.v[j], both(r.inv), both(kMagic));
    const float2 d = fma2(a.v[j], both(-r.inv), add2(m, both(-kMagic)));
    n[2 * j] = __float_as_uint(m.x);
    n[2 * j + 1] = __float_as_uint(m.y);
    off[2 * j] = d.x;
    off[2 * j + 1] = d.y;
    worst = max_magnitude(worst, d.x, d.y);
  }
  if (!(worst <= r.safe)) {
#pragma unroll
    for (int j = 0; j < R::V; ++j)
      if (!(fabsf(off[j]) <= r.safe)) n[j] = quantize_exact(a[j], r.big);
  }
  if (!r.finite) {
#pragma unroll
    for (int j = 0; j < R::V; ++j) n[j] = 0u;
  }
  if constexpr (SG == 0) {
    uint32_t w[R::V / 4];
#pragma unroll
    for (int j = 0; j < R::V / 4; ++j)
      w[j] = __byte_perm(__byte_perm(n[4 * j], n[4 * j + 1], 0x0040),
                         __byte_perm(n[4 * j + 2], n[4 * j + 3], 0x0040), 0x5410);
    const int c = R::col(t, i, 0, G);
    if (c >= K) return;
    if constexpr (R::V == 4) *reinterpret_cast<uint32_t*>(row + c) = w[0];
    else *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = R::col(t, i, j, G);
      if (c < K) row[c] = static_cast<int8_t>(n[j]);
    }
  }
}

// ---------------------------------------------------------------- reductions over a row
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct RowSums {  // two: a warp may be a row ahead of the warps that still read the last row's
  float sum[2][32];
  uint32_t top[2][32];
};

// Sum and bit-pattern maximum over the warp or (s != null) the block, the same on every thread.
template <bool SUM, bool TOP>
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& top, RowSums* s, int flip) {
  if constexpr (SUM) sum = warp_sum(sum);
  if constexpr (TOP) top = __reduce_max_sync(0xffffffffu, top);
  if (s == nullptr) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) {
    if constexpr (SUM) s->sum[flip][warp] = sum;
    if constexpr (TOP) s->top[flip][warp] = top;
  }
  __syncthreads();
  if constexpr (SUM) sum = warp_sum(lane < warps ? s->sum[flip][lane] : 0.f);
  if constexpr (TOP) top = __reduce_max_sync(0xffffffffu, lane < warps ? s->top[flip][lane] : 0u);
}

__device__ __forceinline__ float rstd_of(float sum_squares, int K, float eps) {
  return __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum_squares, static_cast<float>(K)), eps)));
}

// ---------------------------------------------------------------- rows through shared memory
// The kernels for many rows walk over them with a ring of row buffers, filled by bulk copies that
// run ahead of the arithmetic: the copies need no registers, so several rows per block are on
// their way whatever the arithmetic and its barrier do. A buffer is free again once the block has
// passed the row's reduction, behind which every thread holds its elements in registers.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

constexpr int kMaxStages = 8;

struct RowRing {
  uint64_t full[kMaxStages];
};

// Fault path: the copies of the row whose wait gave up and of those after it land (or not, which
// is bounded) before the block's shared memory is given back.
__device__ __forceinline__ void settle_rows(RowRing& ring, int stages, int s, uint32_t ph, int64_t row, int64_t M) {
  for (int i = 0; i < stages && row < M; ++i, row += gridDim.x) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(&ring.full[s], ph) && globaltimer_ns() - t0 < C3CU_WAIT_LIMIT_NS / 16) {
    }
    if (++s == stages) { s = 0; ph ^= 1u; }
  }
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
  int stages;           // ring kernel
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

// The largest magnitudes of eight bf16 as they lie in memory, two at a time (a NaN if there is one).
__device__ __forceinline__ void max_magnitude8(const uint4& w, __nv_bfloat162& top) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x[j])));
}

// One run of a row: the sum of squares and the largest |a|; a = h * w replaces h.
template <bool NORM, int V>
__device__ __forceinline__ void accumulate(Run<V>& a, const Run<V>& w, float2& squares, float& top) {
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {
    if constexpr (NORM) {
      squares = fma2(a.v[j], a.v[j], squares);
      a.v[j] = mul2(a.v[j], w.v[j]);
    }
    top = max_magnitude(top, a.v[j].x, a.v[j].y);
  }
}

// One row per block (or, with 32 threads a row, per warp), held in registers between the reduction
// and the rounding.
template <typename T, bool NORM, bool RES, int SG, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) rows_kernel(const FwdArgs p) {
  using R = Runs<T, SG>;
  constexpr int N = kRowElems / R::V;
  __shared__ RowSums sums;
  const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)
                           : static_cast<int64_t>(blockIdx.x);
  if (WARP && row >= p.M) return;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int G = WARP ? 32 : blockDim.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  Run<R::V> a[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (R::any(t, i, G, p.K)) load<T, SG>(x, t, i, G, p.K, a[i]);
    else clear(a[i]);
  }
  if constexpr (RES) {
    const T* r = static_cast<const T*>(p.res) + row * p.ldr;
    T* h = static_cast<T*>(p.h) + row * p.ldh;
    Run<R::V> b[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (R::any(t, i, G, p.K)) load<T, SG>(r, t, i, G, p.K, b[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (R::any(t, i, G, p.K)) {
#pragma unroll
        for (int j = 0; j < R::V / 2; ++j) a[i].v[j] = add2(a[i].v[j], b[i].v[j]);
        store<T, SG>(h, t, i, G, p.K, a[i]);
      }
    }
  }
  float2 squares = make_float2(0.f, 0.f);
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (R::any(t, i, G, p.K)) {
      Run<R::V> w;
      if constexpr (NORM) load_weight<T, SG>(p.weight, t, i, G, p.K, w);
      accumulate<NORM, R::V>(a[i], w, squares, big);
    }
  }
  float sum = squares.x + squares.y;
  uint32_t top = __float_as_uint(big);
  row_reduce<NORM, true>(sum, top, WARP ? nullptr : &sums, 0);
  const RowScale r = row_scale(top);
  int8_t* q = p.q + row * p.ldq;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (R::any(t, i, G, p.K)) store_q<T, SG>(q, t, i, G, p.K, a[i], r);
  if (t == 0) row_outputs(p, row, sum, r, NORM);
}

// The same over many rows, grid-strided, through the ring (16-byte rows only).
template <typename T, bool NORM, bool RES, int N>
__global__ void __launch_bounds__(1024) ring_rows_kernel(const FwdArgs p) {
  constexpr int V = Runs<T, 0>::V;
  extern __shared__ __align__(128) uint8_t rows[];
  __shared__ RowSums sums;
  __shared__ RowRing ring;
  const int t = threadIdx.x, G = blockDim.x;
  const uint32_t bytes = static_cast<uint32_t>(p.K) * sizeof(T);
  const uint32_t stage = (RES ? 2u : 1u) * bytes;
  auto fill = [&](int s, int64_t row) {
    mbar_arrive_expect_tx(&ring.full[s], stage);
    bulk_load(rows + s * stage, static_cast<const T*>(p.x) + row * p.ldx, bytes, &ring.full[s]);
    if constexpr (RES) bulk_load(rows + s * stage + bytes, static_cast<const T*>(p.res) + row * p.ldr, bytes, &ring.full[s]);
  };
  if (t == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&ring.full[s], 1);
    fence_mbarrier_init();
    fence_proxy_async_shared();
    for (int s = 0; s < p.stages; ++s) {
      const int64_t row = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
      if (row < p.M) fill(s, row);
    }
  }
  __syncthreads();
  int s = 0, flip = 0;
  uint32_t ph = 0;
  int64_t row = blockIdx.x;
  for (; row < p.M; row += gridDim.x) {
    if (!mbar_wait(&ring.full[s], ph, kFaultWaitFull)) break;
    const uint4* xs = reinterpret_cast<const uint4*>(rows + s * stage);
    [[maybe_unused]] const uint4* rs = reinterpret_cast<const uint4*>(rows + s * stage + bytes);
    Run<V> a[N];
    float2 squares = make_float2(0.f, 0.f);
    float big = 0.f;
    constexpr bool kPackedMax = !NORM && V == 8;
    [[maybe_unused]] __nv_bfloat162 big2 = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int v = t + i * G, c = v * V;
      if (c < p.K) {
        const uint4 raw = xs[v];
        expand<T>(raw, a[i]);
        if constexpr (RES) {
          Run<V> b;
          expand<T>(rs[v], b);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) a[i].v[j] = add2(a[i].v[j], b.v[j]);
          store<T, 0>(static_cast<T*>(p.h) + row * p.ldh, t, i, G, p.K, a[i]);
        }
        Run<V> w;
        if constexpr (NORM) load_weight<T, 0>(p.weight, t, i, G, p.K, w);
        if constexpr (kPackedMax) max_magnitude8(raw, big2);
        else accumulate<NORM, V>(a[i], w, squares, big);
      }
    }
    if constexpr (kPackedMax) big = max_magnitude(0.f, __low2float(big2), __high2float(big2));
    float sum = squares.x + squares.y;
    uint32_t top = __float_as_uint(big);
    row_reduce<NORM, true>(sum, top, &sums, flip);
    flip ^= 1;
    if (t == 0) {
      const int64_t next = row + static_cast<int64_t>(p.stages) * gridDim.x;
      if (next < p.M) fill(s, next);
    }
    const RowScale r = row_scale(top);
    int8_t* q = p.q + row * p.ldq;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (Runs<T, 0>::any(t, i, G, p.K)) store_q<T, 0>(q, t, i, G, p.K, a[i], r);
    if (t == 0) row_outputs(p, row, sum, r, NORM);
    if (++s == p.stages) { s = 0; ph ^= 1u; }
  }
  if (row < p.M && t == 0) settle_rows(ring, p.stages, s, ph, row, p.M);
}

// Rows too long for the registers of a block: two passes over the row. The second reads x again
// (or h, which each thread wrote itself).
template <typename T, bool NORM, bool RES, int SG>
__global__ void __launch_bounds__(1024) long_rows_kernel(const FwdArgs p) {
  using R = Runs<T, SG>;
  constexpr int V = R::V;
  __shared__ RowSums sums;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, G = blockDim.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* r = RES ? static_cast<const T*>(p.res) + row * p.ldr : nullptr;
  T* h = RES ? static_cast<T*>(p.h) + row * p.ldh : nullptr;
  const int runs = (p.K - 1) / (V * G) + 1;
  float2 squares = make_float2(0.f, 0.f);
  float big = 0.f;
  for (int i = 0; i < runs; ++i) {
    Run<V> a, w;
    load<T, SG>(x, t, i, G, p.K, a);
    if constexpr (RES) {
      Run<V> b;
      load<T, SG>(r, t, i, G, p.K, b);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) a.v[j] = add2(a.v[j], b.v[j]);
      store<T, SG>(h, t, i, G, p.K, a);
    }
    if constexpr (NORM) load_weight<T, SG>(p.weight, t, i, G, p.K, w);
    accumulate<NORM, V>(a, w, squares, big);
  }
  float sum = squares.x + squares.y;
  uint32_t top = __float_as_uint(big);
  row_reduce<NORM, true>(sum, top, &sums, 0);
  const RowScale rs = row_scale(top);
  int8_t* q = p.q + row * p.ldq;
  const T* again = RES ? h : x;
  for (int i = 0; i < runs; ++i) {
    Run<V> a;
    load<T, SG>(again, t, i, G, p.K, a);
    if constexpr (NORM) {
      Run<V> w;
      load_weight<T, SG>(p.weight, t, i, G, p.K, w);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) a.v[j] = mul2(a.v[j], w.v[j]);
    }
    store_q<T, SG>(q, t, i, G, p.K, a, rs);
  }
  if (t == 0) row_outputs(p, row, sum, rs, NORM);
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
  int stages;      // ring form
};

// g = w dy, xhat = h rstd: dx = rstd (g - xhat mean(g xhat)) + dh, dweight = sum_rows dy xhat.
// A block walks over rows (grid-strided); a thread owns the same N runs of columns in each, so
// dweight's share of the block stays in registers until the end. RING: rows come through the ring
// of buffers (16-byte rows only); else straight from global memory.
template <typename T, bool RING, int SG>
__global__ void __launch_bounds__(512) norm_bwd_kernel(const BwdArgs p) {
  using R = Runs<T, SG>;
  constexpr int V = R::V, N = kRowElems / V;
  extern __shared__ __align__(128) uint8_t rows[];
  __shared__ RowSums sums;
  __shared__ RowRing ring;
  const int t = threadIdx.x, G = blockDim.x;
  const uint32_t bytes = static_cast<uint32_t>(p.K) * sizeof(T);
  const uint32_t stage = (p.dh ? 3u : 2u) * bytes;
  auto fill = [&](int s, int64_t row) {
    mbar_arrive_expect_tx(&ring.full[s], stage);
    uint8_t* to = rows + s * stage;
    bulk_load(to, static_cast<const T*>(p.dy) + row * p.ldy, bytes, &ring.full[s]);
    bulk_load(to + bytes, static_cast<const T*>(p.h) + row * p.ldhh, bytes, &ring.full[s]);
    if (p.dh) bulk_load(to + 2 * bytes, static_cast<const T*>(p.dh) + row * p.lddh, bytes, &ring.full[s]);
  };
  if constexpr (RING) {
    if (t == 0) {
      for (int s = 0; s < p.stages; ++s) mbar_init(&ring.full[s], 1);
      fence_mbarrier_init();
      fence_proxy_async_shared();
      for (int s = 0; s < p.stages; ++s) {
        const int64_t row = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
        if (row < p.M) fill(s, row);
      }
    }
  }
  Run<V> w[N], acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    clear(acc[i]);
    if (R::any(t, i, G, p.K)) load_weight<T, SG>(p.weight, t, i, G, p.K, w[i]);
    else clear(w[i]);
  }
  const float inv_k = __fdiv_rn(1.f, static_cast<float>(p.K));
  if constexpr (RING) __syncthreads();
  int s = 0, flip = 0;
  uint32_t ph = 0;
  int64_t row = blockIdx.x;
  for (; row < p.M; row += gridDim.x) {
    const float rs = __ldg(p.rstd + row);
    Run<V> g[N], xh[N], d[N];
    if constexpr (RING) {
      if (!mbar_wait(&ring.full[s], ph, kFaultWaitFull)) break;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      clear(g[i]);
      clear(xh[i]);
      clear(d[i]);
      if (R::any(t, i, G, p.K)) {
        if constexpr (RING) {
          const uint4* from = reinterpret_cast<const uint4*>(rows + s * stage) + (t + i * G);
          expand<T>(from[0], g[i]);
          expand<T>(from[bytes / 16], xh[i]);
          if (p.dh) expand<T>(from[2 * (bytes / 16)], d[i]);
        } else {
          load<T, SG>(static_cast<const T*>(p.dy) + row * p.ldy, t, i, G, p.K, g[i]);
          load<T, SG>(static_cast<const T*>(p.h) + row * p.ldhh, t, i, G, p.K, xh[i]);
          if (p.dh) load<T, SG>(static_cast<const T*>(p.dh) + row * p.lddh, t, i, G, p.K, d[i]);
        }
      }
    }
    float2 dots = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        xh[i].v[j] = mul2(xh[i].v[j], both(rs));
        acc[i].v[j] = fma2(g[i].v[j], xh[i].v[j], acc[i].v[j]);
        g[i].v[j] = mul2(g[i].v[j], w[i].v[j]);
        dots = fma2(g[i].v[j], xh[i].v[j], dots);
      }
    float dot = dots.x + dots.y;
    uint32_t unused = 0u;
    row_reduce<true, false>(dot, unused, &sums, flip);
    flip ^= 1;
    if constexpr (RING) {
      if (t == 0) {
        const int64_t next = row + static_cast<int64_t>(p.stages) * gridDim.x;
        if (next < p.M) fill(s, next);
      }
      if (++s == p.stages) { s = 0; ph ^= 1u; }
    }
    dot *= -inv_k;
    T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (R::any(t, i, G, p.K)) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j)
          d[i].v[j] = fma2(both(rs), fma2(xh[i].v[j], both(dot), g[i].v[j]), d[i].v[j]);
        store<T, SG>(dx, t, i, G, p.K, d[i]);
      }
    }
  }
  if (RING && row < p.M && t == 0) settle_rows(ring, p.stages, s, ph, row, p.M);
  float* out = gridDim.x == 1 ? p.dweight : p.partial + static_cast<int64_t>(blockIdx.x) * p.K;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (R::any(t, i, G, p.K)) store_sums<T, SG>(out, t, i, G, p.K, acc[i]);
}

// Long rows: the rows' dot products first, then dx and dweight by strips of columns.
constexpr int kStripThreads = 128;

template <typename T, int SG>
__global__ void __launch_bounds__(512) norm_bwd_dot_kernel(const BwdArgs p, float* __restrict__ dots) {
  constexpr int V = Runs<T, SG>::V;
  __shared__ RowSums sums;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, G = blockDim.x;
  const T* dy = static_cast<const T*>(p.dy) + row * p.ldy;
  const T* h = static_cast<const T*>(p.h) + row * p.ldhh;
  const float rs = __ldg(p.rstd + row);
  float2 acc = make_float2(0.f, 0.f);
  const int runs = (p.K - 1) / (V * G) + 1;
#pragma unroll 2
  for (int i = 0; i < runs; ++i) {
    Run<V> g, x, w;
    load<T, SG>(dy, t, i, G, p.K, g);
    load<T, SG>(h, t, i, G, p.K, x);
    load_weight<T, SG>(p.weight, t, i, G, p.K, w);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) acc = fma2(mul2(g.v[j], w.v[j]), mul2(x.v[j], both(rs)), acc);
  }
  float dot = acc.x + acc.y;
  uint32_t unused = 0u;
  row_reduce<true, false>(dot, unused, &sums, 0);
  if (t == 0) dots[row] = dot / static_cast<float>(p.K);
}

// A thread takes one run of columns over `rows_per_block` rows.
template <typename T, int SG>
__global__ void __launch_bounds__(kStripThreads) norm_bwd_strip_kernel(const BwdArgs p, const float* __restrict__ dots,
                                                                       int rows_per_block) {
  constexpr int V = Runs<T, SG>::V;
  const int t = threadIdx.x, G = blockDim.x;
  const int c0 = static_cast<int>(blockIdx.x) * (kStripThreads * V);  // the strip's first column
  const int K = p.K - c0;
  if (!Runs<T, SG>::any(t, 0, G, K)) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t r1 = min(r0 + rows_per_block, static_cast<int64_t>(p.M));
  Run<V> w, acc;
  clear(acc);
  load_weight<T, SG>(p.weight + c0, t, 0, G, K, w);
#pragma unroll 2
  for (int64_t row = r0; row < r1; ++row) {
    Run<V> g, x, d;
    load<T, SG>(static_cast<const T*>(p.dy) + row * p.ldy + c0, t, 0, G, K, g);
    load<T, SG>(static_cast<const T*>(p.h) + row * p.ldhh + c0, t, 0, G, K, x);
    clear(d);
    if (p.dh) load<T, SG>(static_cast<const T*>(p.dh) + row * p.lddh + c0, t, 0, G, K, d);
    const float rs = __ldg(p.rstd + row), dot = -dots[row];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 xh = mul2(x.v[j], both(rs));
      acc.v[j] = fma2(g.v[j], xh, acc.v[j]);
      d.v[j] = fma2(both(rs), fma2(xh, both(dot), mul2(g.v[j], w.v[j])), d.v[j]);
    }
    store<T, SG>(static_cast<T*>(p.dx) + row * p.lddx + c0, t, 0, G, K, d);
  }
  store_sums<T, SG>((gridDim.y == 1 ? p.dweight : p.partial + static_cast<int64_t>(blockIdx.y) * p.K) + c0, t, 0, G, K,
                    acc);
}

// dweight = sum of the blocks' shares, in a fixed order.
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* __restrict__ partial, float* __restrict__ out,
                                                            int rows, int K) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int warp = threadIdx.x >> 5;
  float acc = 0.f;
  if (c < K) {
#pragma unroll 8
    for (int r = warp; r < rows; r += 32) acc += __ldcs(partial + static_cast<int64_t>(r) * K + c);
  }
  __shared__ float part[32][33];
  part[warp][threadIdx.x & 31] = acc;
  __syncthreads();
  acc = warp_sum(part[threadIdx.x & 31][warp]);  // warp w: column w of the strip
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * 32 + warp;
  if ((threadIdx.x & 31) == 0 && mine < K) out[mine] = acc;
}

// ---------------------------------------------------------------- launch rules
inline bool rows_aligned(const void* p, int64_t ld, int64_t M, int esize, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (M <= 1 || ld * esize % bytes == 0);
}

constexpr int kRegRow = kRowElems * 1024;      // the longest row a block holds in registers
constexpr int kRingSmem = 220 * 1024;          // shared memory per SM that rings may take together

// Blocks per SM and ring depth of a kernel of `threads` threads and `regs` registers per thread,
// for rows of `row_bytes` (all inputs of a row). At least two stages, or no ring at all (0).
inline int ring_stages(int threads, int regs, int64_t row_bytes, int* blocks) {
  int per_sm = 65536 / (regs * threads);
  if (per_sm > 2048 / threads) per_sm = 2048 / threads;
  if (per_sm > 16) per_sm = 16;
  for (; per_sm > 0; --per_sm) {
    int64_t stages = (kRingSmem / per_sm - 2048) / row_bytes;
    if (stages > kMaxStages) stages = kMaxStages;
    if (stages >= 2) {
      *blocks = per_sm;
      return static_cast<int>(stages);
    }
  }
  return 0;
}

template <typename T, bool NORM, bool RES, int SG>
cudaError_t launch_rows_sg(const FwdArgs& p, int threads, cudaStream_t st) {
  if (threads <= 32) {
    const int per = 4;
    rows_kernel<T, NORM, RES, SG, true><<<(p.M + per - 1) / per, 32 * per, 0, st>>>(p);
  } else {
    rows_kernel<T, NORM, RES, SG, false><<<p.M, threads, 0, st>>>(p);
  }
  return cudaGetLastError();
}

// 16 elements per thread; a row over 16 * 1024 elements takes two passes.
template <typename T, bool NORM, bool RES>
cudaError_t launch_rows(FwdArgs p, bool vec, cudaStream_t st) {
  if (p.K > kRegRow) {
    if (vec) long_rows_kernel<T, NORM, RES, 0><<<p.M, 1024, 0, st>>>(p);
    else long_rows_kernel<T, NORM, RES, 1024><<<p.M, 1024, 0, st>>>(p);
    return cudaGetLastError();
  }
  if (!vec) {
    if (p.K <= 32 * kRowElems) return launch_rows_sg<T, NORM, RES, 32>(p, 32, st);
    if (p.K <= 128 * kRowElems) return launch_rows_sg<T, NORM, RES, 128>(p, 128, st);
    if (p.K <= 256 * kRowElems) return launch_rows_sg<T, NORM, RES, 256>(p, 256, st);
    if (p.K <= 512 * kRowElems) return launch_rows_sg<T, NORM, RES, 512>(p, 512, st);
    return launch_rows_sg<T, NORM, RES, 1024>(p, 1024, st);
  }
  // Elements per thread: quantising alone is short of issue slots (4096 wide: 243 instructions per
  // warp and row at 16), and twice the elements halve what a row costs besides them.
  constexpr int E = NORM ? kRowElems : 2 * kRowElems;
  const int ring_threads = (p.K + E * 32 - 1) / (E * 32) * 32;
  int per_sm = 0;
  const int64_t row_bytes = static_cast<int64_t>(p.K) * sizeof(T) * (RES ? 2 : 1);
  const int stages = ring_stages(ring_threads, 64, row_bytes, &per_sm);
  const int64_t grid = static_cast<int64_t>(sm_count()) * per_sm;
  const char* e = getenv("DEV_RING");
  if (stages >= 2 && p.M >= 2 * grid && !(e && e[0]=='0')) {
    auto kern = ring_rows_kernel<T, NORM, RES, E / Runs<T, 0>::V>;
    static std::atomic<uint64_t> smem_set{0};
    if (set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kRingSmem, smem_set, "rows: set shared memory") == C3CU_OK) {
      p.stages = stages;
      kern<<<static_cast<unsigned>(grid), ring_threads, static_cast<size_t>(stages * row_bytes), st>>>(p);
      return cudaGetLastError();
    }
  }
  return launch_rows_sg<T, NORM, RES, 0>(p, (p.K + kRowElems * 32 - 1) / (kRowElems * 32) * 32, st);
}

template <typename T>
int fwd(const FwdArgs& p, bool norm, cudaStream_t st, const char* what) {
  constexpr int V = Runs<T, 0>::V;
  const int e = static_cast<int>(sizeof(T));
  bool vec = p.K % V == 0 && rows_aligned(p.x, p.ldx, p.M, e, 16) && rows_aligned(p.q, p.ldq, p.M, 1, V);
  if (norm) vec = vec && aligned16(p.weight);
  if (p.res) vec = vec && rows_aligned(p.res, p.ldr, p.M, e, 16) && rows_aligned(p.h, p.ldh, p.M, e, 16);
  cudaError_t err = !norm ? launch_rows<T, false, false>(p, vec, st)
                   : p.res ? launch_rows<T, true, true>(p, vec, st) : launch_rows<T, true, false>(p, vec, st);
  return cuda_status(err, what);
}

constexpr int kBwdMaxK = 512 * kRowElems;  // beyond: strips

// Rows of a strip block: enough blocks for every SM to have eight, at least 16 rows, and a grid
// whose y dimension keeps its limit.
int strip_rows(int64_t M, int64_t K, int cols) {
  const int64_t strips = (K + cols - 1) / cols;
  const int64_t bands = 148 * 8 / strips > 0 ? 148 * 8 / strips : 1;
  int64_t rows = (M + bands - 1) / bands;
  if (rows < 16) rows = 16;
  if (rows * 65535 < M) rows = (M + 65534) / 65535;
  return static_cast<int>(rows);
}

// Threads of a block: 16 columns each; single elements need a power of two (a kernel for each).
int bwd_threads(int64_t K, bool vec) {
  const int warps = static_cast<int>((K + kRowElems * 32 - 1) / (kRowElems * 32));
  if (vec) return warps * 32;
  int t = 32;
  while (t < warps * 32) t *= 2;
  return t;
}

// 128 registers a thread: 512 threads per SM.
int bwd_blocks_per_sm(int threads) { return 512 / threads < 16 ? 512 / threads : 16; }

// Rows of partial sums, one a block; `cols`: a strip's columns.
size_t bwd_partial_rows(int64_t M, int64_t K, bool vec, int cols) {
  if (K <= kBwdMaxK) {
    const int64_t most = static_cast<int64_t>(sm_count() > 0 ? sm_count() : 148) * bwd_blocks_per_sm(bwd_threads(K, vec));
    return static_cast<size_t>(M < most ? M : most);
  }
  const int64_t rows = strip_rows(M, K, cols);
  return static_cast<size_t>((M + rows - 1) / rows);
}

template <typename T>
cudaError_t launch_bwd(BwdArgs p, bool vec, int rows, int threads, cudaStream_t st) {
  if (!vec) {
    switch (threads) {
      case 32: norm_bwd_kernel<T, false, 32><<<rows, 32, 0, st>>>(p); break;
      case 64: norm_bwd_kernel<T, false, 64><<<rows, 64, 0, st>>>(p); break;
      case 128: norm_bwd_kernel<T, false, 128><<<rows, 128, 0, st>>>(p); break;
      case 256: norm_bwd_kernel<T, false, 256><<<rows, 256, 0, st>>>(p); break;
      default: norm_bwd_kernel<T, false, 512><<<rows, 512, 0, st>>>(p); break;
    }
    return cudaGetLastError();
  }
  const int64_t row_bytes = static_cast<int64_t>(p.K) * sizeof(T) * (p.dh ? 3 : 2);
  int64_t stages = (kRingSmem / bwd_blocks_per_sm(threads) - 2048) / row_bytes;
  if (stages > kMaxStages) stages = kMaxStages;
  const char* e = getenv("DEV_RING");
  if (stages >= 2 && p.M >= 2 * rows && !(e && e[0] == '0')) {
    auto kern = norm_bwd_kernel<T, true, 0>;
    static std::atomic<uint64_t> smem_set{0};
    if (set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kRingSmem, smem_set,
                             "rms_norm_bwd: set shared memory") == C3CU_OK) {
      p.stages = static_cast<int>(stages);
      kern<<<rows, threads, static_cast<size_t>(stages * row_bytes), st>>>(p);
      return cudaGetLastError();
    }
  }
  norm_bwd_kernel<T, false, 0><<<rows, threads, 0, st>>>(p);
  return cudaGetLastError();
}

template <typename T, int SG>
cudaError_t launch_bwd_strips(BwdArgs p, float* dots, int rows, cudaStream_t st) {
  constexpr int kCols = kStripThreads * Runs<T, SG>::V;
  norm_bwd_dot_kernel<T, SG ? 512 : 0><<<p.M, 512, 0, st>>>(p, dots);
  norm_bwd_strip_kernel<T, SG><<<dim3((p.K + kCols - 1) / kCols, rows), kStripThreads, 0, st>>>(p, dots,
                                                                                            strip_rows(p.M, p.K, kCols));
  return cudaGetLastError();
}

template <typename T>
int bwd(BwdArgs p, bool vec, float* ws, cudaStream_t st) {
  const int cols = kStripThreads * (vec ? Runs<T, 0>::V : 8);
  const int rows = static_cast<int>(bwd_partial_rows(p.M, p.K, vec, cols));
  cudaError_t err;
  if (p.K <= kBwdMaxK) {
    p.partial = ws;
    err = launch_bwd<T>(p, vec, rows, bwd_threads(p.K, vec), st);
  } else {
    p.partial = ws + p.M;
    err = vec ? launch_bwd_strips<T, 0>(p, ws, rows, st) : launch_bwd_strips<T, kStripThreads>(p, ws, rows, st);
  }
  int rc = cuda_status(err, "rms_norm_bwd: launch");
  if (rc != C3CU_OK || rows <= 1) return rc;
  sum_partials_kernel<<<(p.K + 31) / 32, 1024, 0, st>>>(p.partial, p.dweight, rows, p.K);
  return cuda_status(cudaGetLastError(), "rms_norm_bwd: launch");
}

int check_sizes(const char* what, int64_t M, int64_t K, int dtype) {
  if (dtype != C3CU_DTYPE_F32 && dtype != C3CU_DTYPE_BF16) {
    set_error("%s: dtype %d is neither f32 nor bf16", what, dtype);
    return C3CU_ERR_INVALID;
  }
  if (M < 0 || K < 1 || M > INT32_MAX - 65536 || K > INT32_MAX - 65536) {
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
  size_t rows = 1;  // the most that any element type and alignment needs
  for (bool vec : {false, true}) {
    for (int v : {4, 8}) {
      const size_t n = quant::bwd_partial_rows(M, K, vec, quant::kStripThreads * v);
      if (n > rows) rows = n;
    }
  }
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
