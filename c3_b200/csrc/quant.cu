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
// launch shape: an element whose fp32 quotient lies too near to a half-integer is decided by the
// sign of 254 a - (2 n + 1) A, which fp32 with fused multiply-adds gives exactly.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "host_util.h"

C3CU_FAULT_ACCESSORS(quant)

namespace c3cu {
namespace quant {

constexpr int kRowElems = 16;  // elements of a row per thread, where a row is held in registers

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
    using Raw = typename std::conditional<sizeof(T) == 4, uint32_t, unsigned short>::type;
    const Raw* from = reinterpret_cast<const Raw*>(row) + t + i * 8 * SG;
    uint32_t f[8];
    if ((i + 1) * 8 * SG <= K) {  // the whole block's runs: no bounds
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = from[j * SG];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = R::col(t, i, j, G) < K ? from[j * SG] : Raw{0};
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] <<= 32 - 8 * sizeof(T);
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = make_float2(__uint_as_float(f[2 * j]), __uint_as_float(f[2 * j + 1]));
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
    const float* from = w + t + i * 8 * SG;
    if ((i + 1) * 8 * SG <= K) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __ldg(from + j * SG);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = R::col(t, i, j, G) < K ? __ldg(from + j * SG) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = make_float2(f[2 * j], f[2 * j + 1]);
  }
}

// Eight elements SG apart, those at columns below K (`to` is column c's address).
template <int SG, typename T>
__device__ __forceinline__ void store_strided(T* to, int c, int K, const T (&f)[8]) {
  if (c + 8 * SG <= K) {
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j * SG] = f[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j * SG < K) to[j * SG] = f[j];
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
    T* to = row + t + i * 8 * SG;
    T f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        f[2 * j] = x.v[j].x;
        f[2 * j + 1] = x.v[j].y;
      } else {
        const uint32_t w = pack_bf16x2(x.v[j].x, x.v[j].y);
        f[2 * j] = __ushort_as_bfloat16(static_cast<unsigned short>(w));
        f[2 * j + 1] = __ushort_as_bfloat16(static_cast<unsigned short>(w >> 16));
        x.v[j] = unpack(w);
      }
    }
    store_strided<SG>(to, t + i * 8 * SG, K, f);
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
struct RowScale {
  float big;   // A
  float inv;   // 127 / A, within 2^-24 of it: an approximate reciprocal and one step of Newton's method
  float safe;  // largest |a inv - round(a inv)| at which a inv rounds like the real quotient
  bool finite, tame;
};

// `bits` is the largest |a| as its bit pattern (which orders like the number, with infinities and
// NaN on top).
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale r;
  r.big = __uint_as_float(bits);
  r.finite = bits < 0x7f800000u;
  // Beyond this range 127 / A or 254 a could leave fp32's: such rows take fp64 divisions.
  r.tame = r.big > 1e-25f && r.big < 1e35f;
  float rcp;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rcp) : "f"(r.big));
  const float inv = 127.f * rcp;
  r.inv = r.tame ? fmaf(fmaf(-inv, r.big, 127.f), rcp, inv) : 0.f;
  // a inv, multiplied without a rounding, is off by inv's error: at most 127 * 2^-23
  r.safe = 0.5f - 1.6e-5f;
  return r;
}

// The nearest integer to 127 a / A, ties to even, given one of its two neighbours n = round(a inv)
// and off = a inv - n, near +-1/2: whether the quotient is beyond the half-integer b / 2,
// b = 2 n +- 1, is the sign of 254 a - b A. Both products are taken apart into their rounded value
// and the rest (exact, 32 bits each); the values are so near each other that they subtract exactly.
__device__ __forceinline__ float decide(float a, float big, float n, float off) {
  const float way = off > 0.f ? 1.f : -1.f;
  const float b = fmaf(2.f, n, way);
  const float p = __fmul_rn(254.f, a), q = __fmul_rn(b, big);
  const float rest = __fsub_rn(fmaf(254.f, a, -p), fmaf(b, big, -q));
  const float diff = __fmul_rn(__fadd_rn(__fsub_rn(p, q), rest), way);
  const bool odd = static_cast<int>(n) & 1;
  return diff > 0.f || (diff == 0.f && odd) ? n + way : n;
}

// A row of extreme magnitude.
__device__ __noinline__ float quantize_wild(float a, float big) {
  return big > 0.f ? static_cast<float>(rint(127.0 * static_cast<double>(a) / static_cast<double>(big))) : 0.f;
}

template <typename T, int SG>
__device__ __forceinline__ void store_q(int8_t* row, int t, int i, int G, int K, const Run<Runs<T, SG>::V>& a,
                                        const RowScale& r) {
  using R = Runs<T, SG>;
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it leaves round(a inv) in the low bits
  float m[R::V], off[R::V];
  float worst = 0.f;
#pragma unroll
  for (int j = 0; j < R::V / 2; ++j) {
    const float2 x = fma2(a.v[j], both(r.inv), both(kMagic));
    const float2 d = fma2(a.v[j], both(r.inv), add2(both(kMagic), make_float2(-x.x, -x.y)));
    m[2 * j] = x.x;
    m[2 * j + 1] = x.y;
    off[2 * j] = d.x;
    off[2 * j + 1] = d.y;
    worst = max_magnitude(worst, d.x, d.y);
  }
  if (worst > r.safe) {
#pragma unroll
    for (int j = 0; j < R::V; ++j)
      if (fabsf(off[j]) > r.safe) m[j] = decide(a[j], r.big, m[j] - kMagic, off[j]) + kMagic;
  }
  if (!r.tame) {
#pragma unroll
    for (int j = 0; j < R::V; ++j) m[j] = (r.finite ? quantize_wild(a[j], r.big) : 0.f) + kMagic;
  }
  uint32_t n[R::V];
#pragma unroll
  for (int j = 0; j < R::V; ++j) n[j] = __float_as_uint(m[j]);
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
    int8_t f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = static_cast<int8_t>(n[j]);
    store_strided<SG>(row + t + i * 8 * SG, t + i * 8 * SG, K, f);
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

// 0 for a row of zeros with eps 0, not infinity, which times the row's zeros would be NaN in the scale, in
// the gradient and so in all of dweight and dW.
__device__ __forceinline__ float rstd_of(float sum_squares, int K, float eps) {
  const float mean = __fadd_rn(__fdiv_rn(sum_squares, static_cast<float>(K)), eps);
  return mean == 0.f ? 0.f : __fdiv_rn(1.f, __fsqrt_rn(mean));
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

// What a bulk copy brings of a row that need not start on 16 bytes: whole 16-byte pieces around it.
// The first and last rows' may reach past the matrix; those rows are read from global memory.
struct Span {
  const uint8_t* from;  // 16-byte aligned
  uint32_t size;        // multiple of 16
  uint32_t skip;        // bytes before the row's first
  bool direct;
};

template <typename T>
__device__ __forceinline__ Span row_span(const void* base, int64_t ld, int M, int64_t row, uint32_t bytes) {
  const uint8_t* first = static_cast<const uint8_t*>(base);
  const uint8_t* start = first + row * ld * static_cast<int64_t>(sizeof(T));
  const uint8_t* end = first + (M - 1) * ld * static_cast<int64_t>(sizeof(T)) + bytes;
  Span r;
  r.skip = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(start) & 15u);
  r.from = start - r.skip;
  r.size = (r.skip + bytes + 15u) & ~15u;
  r.direct = r.from < first || r.from + r.size > end;
  return r;
}

// Bytes of a ring stage that one input's row takes.
__host__ __device__ inline uint32_t row_pitch(uint32_t bytes, bool aligned) {
  return aligned ? bytes : ((bytes + 15u) & ~15u) + 16u;
}

struct RowRing {
  uint64_t full[kMaxStages];
};

// A warp gives up as a whole: the reductions below shuffle between all of its lanes.
__device__ __forceinline__ bool wait_row(RowRing& ring, int s, uint32_t ph) {
  return __all_sync(0xffffffffu, mbar_wait(&ring.full[s], ph, kFaultWaitFull));
}

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
// and the rounding. For few rows, where the launch is most of the time (a token of 4096 with the norm:
// 2.2 us in a graph, an empty kernel 2.1).
template <typename T, bool NORM, bool RES, int SG, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) rows_kernel(const FwdArgs p) {
  using R = Runs<T, SG>;
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

// The same over many rows, grid-strided, through the ring. 16384 x 4096 bf16: norm with residual 76.5
// us (6.1 TB/s; a block a row 88), quantising alone 41 us (4.9 TB/s, a block a row 57), which the issue
// slots bound: the rounding costs about fifteen instructions an element.
template <typename T, bool NORM, bool RES, int SG, int N>
__global__ void __launch_bounds__(1024) ring_rows_kernel(const FwdArgs p) {
  using R = Runs<T, SG>;
  constexpr int V = R::V;
  extern __shared__ __align__(128) uint8_t rows[];
  __shared__ RowSums sums;
  __shared__ RowRing ring;
  const int t = threadIdx.x, G = blockDim.x;
  const uint32_t bytes = static_cast<uint32_t>(p.K) * sizeof(T);
  const uint32_t pitch = row_pitch(bytes, SG == 0);
  const uint32_t stage = (RES ? 2u : 1u) * pitch;
  auto fill = [&](int s, int64_t row) {
    uint8_t* to = rows + s * stage;
    if constexpr (SG == 0) {
      mbar_arrive_expect_tx(&ring.full[s], stage);
      bulk_load(to, static_cast<const T*>(p.x) + row * p.ldx, bytes, &ring.full[s]);
      if constexpr (RES) bulk_load(to + pitch, static_cast<const T*>(p.res) + row * p.ldr, bytes, &ring.full[s]);
    } else {
      const Span x = row_span<T>(p.x, p.ldx, p.M, row, bytes);
      Span r = x;
      if constexpr (RES) r = row_span<T>(p.res, p.ldr, p.M, row, bytes);
      mbar_arrive_expect_tx(&ring.full[s], (x.direct ? 0u : x.size) + (RES && !r.direct ? r.size : 0u));
      if (!x.direct) bulk_load(to, x.from, x.size, &ring.full[s]);
      if (RES && !r.direct) bulk_load(to + pitch, r.from, r.size, &ring.full[s]);
    }
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
    if (!wait_row(ring, s, ph)) break;
    const uint8_t* at = rows + s * stage;
    Run<V> a[N];
    float2 squares = make_float2(0.f, 0.f);
    float big = 0.f;
    constexpr bool kPackedMax = !NORM && SG == 0 && V == 8;
    [[maybe_unused]] __nv_bfloat162 big2 = __floats2bfloat162_rn(0.f, 0.f);
    if constexpr (SG != 0) {
      auto read = [&](const void* base, int64_t ld, const uint8_t* here, Run<V>(&v)[N]) {
        const Span sp = row_span<T>(base, ld, p.M, row, bytes);
        if (sp.direct) {
#pragma unroll
          for (int i = 0; i < N; ++i) load<T, SG>(static_cast<const T*>(base) + row * ld, t, i, G, p.K, v[i]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) load<T, SG>(reinterpret_cast<const T*>(here + sp.skip), t, i, G, p.K, v[i]);
        }
      };
      read(p.x, p.ldx, at, a);
      if constexpr (RES) {
        Run<V> b[N];
        read(p.res, p.ldr, at + pitch, b);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < V / 2; ++j) a[i].v[j] = add2(a[i].v[j], b[i].v[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (R::any(t, i, G, p.K)) {
        if constexpr (SG == 0) {
          const uint4 raw = reinterpret_cast<const uint4*>(at)[t + i * G];
          expand<T>(raw, a[i]);
          if constexpr (kPackedMax) max_magnitude8(raw, big2);
          if constexpr (RES) {
            Run<V> b;
            expand<T>(reinterpret_cast<const uint4*>(at + pitch)[t + i * G], b);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) a[i].v[j] = add2(a[i].v[j], b.v[j]);
          }
        }
        if constexpr (RES) store<T, SG>(static_cast<T*>(p.h) + row * p.ldh, t, i, G, p.K, a[i]);
        Run<V> w;
        if constexpr (NORM) load_weight<T, SG>(p.weight, t, i, G, p.K, w);
        if constexpr (!kPackedMax) accumulate<NORM, V>(a[i], w, squares, big);
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
      if (R::any(t, i, G, p.K)) store_q<T, SG>(q, t, i, G, p.K, a[i], r);
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

// Asks for a row of dy, h and dh, `pitch` apart from `to` on, and arms `bar` with their bytes. Off the
// 16-byte grid the rows that would reach past their matrix are left out.
template <typename T, int SG>
__device__ __forceinline__ void fill_bwd_row(const BwdArgs& p, uint8_t* to, uint64_t* bar, int64_t row, uint32_t bytes,
                                             uint32_t pitch) {
  if constexpr (SG == 0) {
    mbar_arrive_expect_tx(bar, (p.dh ? 3u : 2u) * pitch);
    bulk_load(to, static_cast<const T*>(p.dy) + row * p.ldy, bytes, bar);
    bulk_load(to + pitch, static_cast<const T*>(p.h) + row * p.ldhh, bytes, bar);
    if (p.dh) bulk_load(to + 2 * pitch, static_cast<const T*>(p.dh) + row * p.lddh, bytes, bar);
  } else {
    Span sp[3];
    sp[0] = row_span<T>(p.dy, p.ldy, p.M, row, bytes);
    sp[1] = row_span<T>(p.h, p.ldhh, p.M, row, bytes);
    sp[2] = row_span<T>(p.dh, p.lddh, p.M, row, bytes);
    if (!p.dh) sp[2].direct = true;
    uint32_t tx = 0u;
#pragma unroll
    for (int k = 0; k < 3; ++k) tx += sp[k].direct ? 0u : sp[k].size;
    mbar_arrive_expect_tx(bar, tx);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (!sp[k].direct) bulk_load(to + k * pitch, sp[k].from, sp[k].size, bar);
  }
}

// g = w dy, xhat = h rstd: dx = rstd (g - xhat mean(g xhat)) + dh, dweight = sum_rows dy xhat.
// A block walks over rows (grid-strided); a thread owns the same N runs of columns in each, so
// dweight's share of the block stays in registers until the end. RING: rows come through the ring
// of buffers; else straight from global memory. 16384 x 4096 bf16 with dh: 88.5 us with the sum of the
// shares (6.1 TB/s), 124 without the ring.
template <typename T, bool RING, int SG>
__global__ void __launch_bounds__(512) norm_bwd_kernel(const BwdArgs p) {
  using R = Runs<T, SG>;
  constexpr int V = R::V, N = kRowElems / V;
  extern __shared__ __align__(128) uint8_t rows[];
  __shared__ RowSums sums;
  __shared__ RowRing ring;
  const int t = threadIdx.x, G = blockDim.x;
  const uint32_t bytes = static_cast<uint32_t>(p.K) * sizeof(T);
  const uint32_t pitch = row_pitch(bytes, SG == 0);
  const uint32_t stage = (p.dh ? 3u : 2u) * pitch;
  pdl_launch_dependents();
  auto fill = [&](int s, int64_t row) { fill_bwd_row<T, SG>(p, rows + s * stage, &ring.full[s], row, bytes, pitch); };
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
    const T* from[3] = {static_cast<const T*>(p.dy) + row * p.ldy, static_cast<const T*>(p.h) + row * p.ldhh,
                        p.dh ? static_cast<const T*>(p.dh) + row * p.lddh : nullptr};
    if constexpr (RING) {
      if (!wait_row(ring, s, ph)) break;
    }
    auto read = [&](int k, const void* base, int64_t ld, Run<V>(&v)[N]) {
      bool buffered = RING;
      uint32_t skip = 0u;
      if constexpr (RING && SG != 0) {
        const Span sp = row_span<T>(base, ld, p.M, row, bytes);
        buffered = !sp.direct;
        skip = sp.skip;
      }
      const uint8_t* here = rows + s * stage + k * pitch + skip;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        clear(v[i]);
        if (R::any(t, i, G, p.K)) {
          if constexpr (RING && SG == 0) {
            expand<T>(reinterpret_cast<const uint4*>(here)[t + i * G], v[i]);
          } else {
            if (buffered) load<T, SG>(reinterpret_cast<const T*>(here), t, i, G, p.K, v[i]);
            else load<T, SG>(from[k], t, i, G, p.K, v[i]);
          }
        }
      }
    };
    read(0, p.dy, p.ldy, g);
    read(1, p.h, p.ldhh, xh);
    if (p.dh) {
      read(2, p.dh, p.lddh, d);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) clear(d[i]);
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

// Rows of up to twice that length: 32 columns a thread, of which only dweight's
// shares and the weights fit in registers. So each row is read twice from its buffer, for the dot
// product and for dx, and the buffer is filled again behind the next row's reduction. Against strips,
// which read dy and h twice from HBM, 5461 x 12288 bf16 took 96 us instead of 148 (83 at the copy rate),
// and off the 16-byte grid 5461 x 12287 130 instead of 293.
constexpr int kWideElems = 2 * kRowElems;
constexpr int kWideThreads = 512;

template <typename T, int SG>
__global__ void __launch_bounds__(kWideThreads) norm_bwd_wide_kernel(const BwdArgs p) {
  using R = Runs<T, SG>;
  constexpr int V = R::V, N = kWideElems / V;
  extern __shared__ __align__(128) uint8_t rows[];
  __shared__ RowSums sums;
  __shared__ RowRing ring;
  const int t = threadIdx.x, G = kWideThreads;
  const uint32_t bytes = static_cast<uint32_t>(p.K) * sizeof(T);
  const uint32_t pitch = row_pitch(bytes, SG == 0);
  const uint32_t stage = (p.dh ? 3u : 2u) * pitch;
  pdl_launch_dependents();
  auto fill = [&](int s, int64_t row) { fill_bwd_row<T, SG>(p, rows + s * stage, &ring.full[s], row, bytes, pitch); };
  if (t == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&ring.full[s], 1);
    fence_mbarrier_init();
    fence_proxy_async_shared();
    for (int s = 0; s < p.stages; ++s) {
      const int64_t row = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
      if (row < p.M) fill(s, row);
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
  __syncthreads();
  int s = 0, flip = 0, last = -1;  // last: the buffer of the row before
  uint32_t ph = 0;
  int64_t row = blockIdx.x;
  for (; row < p.M; row += gridDim.x) {
    const float rs = __ldg(p.rstd + row);
    if (!wait_row(ring, s, ph)) break;
    // where the k-th input's row is: in its buffer, or (off the grid, the first and last) where it was
    auto source = [&](int k, const void* base, int64_t ld) {
      const uint8_t* at = rows + s * stage + k * pitch;
      if constexpr (SG == 0) {
        return reinterpret_cast<const T*>(at);
      } else {
        const Span sp = row_span<T>(base, ld, p.M, row, bytes);
        return sp.direct ? static_cast<const T*>(base) + row * ld : reinterpret_cast<const T*>(at + sp.skip);
      }
    };
    auto read = [&](const T* from, int i, Run<V>& v) {
      if constexpr (SG == 0) expand<T>(reinterpret_cast<const uint4*>(from)[t + i * G], v);
      else load<T, SG>(from, t, i, G, p.K, v);
    };
    const T* dy = source(0, p.dy, p.ldy);
    const T* h = source(1, p.h, p.ldhh);
    const T* dh = p.dh ? source(2, p.dh, p.lddh) : nullptr;
    float2 dots = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!R::any(t, i, G, p.K)) continue;
      Run<V> g, xh;
      read(dy, i, g);
      read(h, i, xh);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        xh.v[j] = mul2(xh.v[j], both(rs));
        acc[i].v[j] = fma2(g.v[j], xh.v[j], acc[i].v[j]);
        dots = fma2(mul2(g.v[j], w[i].v[j]), xh.v[j], dots);
      }
    }
    float dot = dots.x + dots.y;
    uint32_t unused = 0u;
    row_reduce<true, false>(dot, unused, &sums, flip);
    flip ^= 1;
    if (t == 0 && last >= 0) {
      const int64_t next = row + static_cast<int64_t>(p.stages - 1) * gridDim.x;
      if (next < p.M) fill(last, next);
    }
    dot *= -inv_k;
    T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!R::any(t, i, G, p.K)) continue;
      Run<V> g, xh, d;
      read(dy, i, g);
      read(h, i, xh);
      clear(d);
      if (p.dh) read(dh, i, d);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        xh.v[j] = mul2(xh.v[j], both(rs));
        d.v[j] = fma2(both(rs), fma2(xh.v[j], both(dot), mul2(g.v[j], w[i].v[j])), d.v[j]);
      }
      store<T, SG>(dx, t, i, G, p.K, d);
    }
    last = s;
    if (++s == p.stages) { s = 0; ph ^= 1u; }
  }
  if (row < p.M && t == 0) settle_rows(ring, p.stages, s, ph, row, p.M);
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * p.K;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (R::any(t, i, G, p.K)) store_sums<T, SG>(out, t, i, G, p.K, acc[i]);
}

// Longer rows, and few: the rows' dot products first, then dx and dweight by strips of columns, so that dy
// and h are read twice.
constexpr int kStripThreads = 128;

template <typename T, int SG>
__global__ void __launch_bounds__(512) norm_bwd_dot_kernel(const BwdArgs p, float* __restrict__ dots) {
  constexpr int V = Runs<T, SG>::V;
  __shared__ RowSums sums;
  pdl_launch_dependents();
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
  pdl_wait();
  pdl_launch_dependents();
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

// dweight = sum of the blocks' shares, in a fixed order. A thread asks for sixteen at a time, those
// past the last among them: rows left over one by one cost a trip to L2 each.
constexpr int kSumAhead = 16;

__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* __restrict__ partial, float* __restrict__ out,
                                                            int rows, int K) {
  pdl_wait();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int warp = threadIdx.x >> 5;
  float acc = 0.f;
  if (c < K) {
    for (int r0 = warp; r0 < rows; r0 += 32 * kSumAhead) {
      float v[kSumAhead];
#pragma unroll
      for (int i = 0; i < kSumAhead; ++i) {
        const int r = r0 + 32 * i;
        v[i] = r < rows ? __ldcs(partial + static_cast<int64_t>(r) * K + c) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kSumAhead; ++i) acc += v[i];
    }
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

template <typename T, bool NORM, bool RES, int SG, int N>
cudaError_t launch_block_rows(const FwdArgs& p, int threads, cudaStream_t st) {
  if (threads <= 32) {
    const int per = 4;
    rows_kernel<T, NORM, RES, SG, N, true><<<(p.M + per - 1) / per, 32 * per, 0, st>>>(p);
  } else {
    rows_kernel<T, NORM, RES, SG, N, false><<<p.M, threads, 0, st>>>(p);
  }
  return cudaGetLastError();
}

// Rows through the ring, if they are many enough for it: at least `times` rows a block.
template <typename T, bool NORM, bool RES, int SG, int N>
bool launch_ring(FwdArgs p, int threads, int times, cudaError_t* err, cudaStream_t st) {
  int per_sm = 0;
  const int64_t row_bytes =
      static_cast<int64_t>(row_pitch(static_cast<uint32_t>(p.K) * sizeof(T), SG == 0)) * (RES ? 2 : 1);
  p.stages = ring_stages(threads, 64, row_bytes, &per_sm);
  const int64_t grid = static_cast<int64_t>(sm_count()) * per_sm;
  if (p.stages < 2 || p.M < times * grid) return false;
  auto kern = ring_rows_kernel<T, NORM, RES, SG, N>;
  static std::atomic<uint64_t> smem_set{0};
  if (set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kRingSmem, smem_set, "rows: set shared memory") != C3CU_OK)
    return false;
  kern<<<static_cast<unsigned>(grid), threads, static_cast<size_t>(p.stages * row_bytes), st>>>(p);
  *err = cudaGetLastError();
  return true;
}

// Rows off the 16-byte grid: 16 or 24 single elements per thread.
template <typename T, bool NORM, bool RES, int SG>
cudaError_t launch_strided(const FwdArgs& p, cudaStream_t st) {
  [[maybe_unused]] cudaError_t err;
  // Single fp32 elements have twice the bytes of bf16 ones in flight, and gain nothing from the ring.
  constexpr bool kRing = sizeof(T) == 2 && SG >= 128;
  if (p.K <= 16 * SG) {
    if constexpr (kRing)
      if (launch_ring<T, NORM, RES, SG, 2>(p, SG, 4, &err, st)) return err;
    return launch_block_rows<T, NORM, RES, SG, 2>(p, SG, st);
  }
  if constexpr (kRing)
    if (launch_ring<T, NORM, RES, SG, 3>(p, SG, 4, &err, st)) return err;
  return launch_block_rows<T, NORM, RES, SG, 3>(p, SG, st);
}

template <typename T, bool NORM, bool RES>
cudaError_t launch_rows(const FwdArgs& p, bool vec, cudaStream_t st) {
  if (p.K > kRegRow) {
    if (vec) long_rows_kernel<T, NORM, RES, 0><<<p.M, 1024, 0, st>>>(p);
    else long_rows_kernel<T, NORM, RES, 1024><<<p.M, 1024, 0, st>>>(p);
    return cudaGetLastError();
  }
  if (!vec) {
    if (p.K <= 24 * 32) return launch_strided<T, NORM, RES, 32>(p, st);
    if (p.K <= 24 * 128) return launch_strided<T, NORM, RES, 128>(p, st);
    if (p.K <= 24 * 256) return launch_strided<T, NORM, RES, 256>(p, st);
    if (p.K <= 24 * 512) return launch_strided<T, NORM, RES, 512>(p, st);
    return launch_strided<T, NORM, RES, 1024>(p, st);
  }
  constexpr int V = Runs<T, 0>::V;
  // The ring pays where a block per row has too little in flight or too few blocks fit: wide rows
  // (us, ring / block per row, bf16, 64 Mi elements: quantise at K 4096 41 / 49, 12288 42 / 69, norm at 4096
  // 77 / 81; but fp32 8192 x 4096 33 / 25), and once its blocks have several rows each. Below 4096 it is
  // either: quantise at K 3584 44 / 49, 2560 49 / 47, 2048 43 / 45, 1536 47 / 45, 1024 55 / 44, norm 74 / 81,
  // 76 / 80, 75 / 77, 80 / 78, 82 / 78.
  if (p.K >= (sizeof(T) == 2 ? 4096 : 8200)) {
    // Elements per thread: quantising alone is short of issue slots, and twice the elements halve
    // what a row costs besides them.
    constexpr int E = NORM ? kRowElems : 2 * kRowElems;
    const int threads = (p.K + E * 32 - 1) / (E * 32) * 32;
    cudaError_t err;
    if (launch_ring<T, NORM, RES, 0, E / V>(p, threads, p.K > 8192 ? 2 : 8, &err, st)) return err;
  }
  return launch_block_rows<T, NORM, RES, 0, kRowElems / V>(p, (p.K + kRowElems * 32 - 1) / (kRowElems * 32) * 32, st);
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

constexpr int kBwdMaxK = 512 * kRowElems;  // beyond: two reads of a buffer, or strips

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
    if (M <= 4) return 1;  // one block walks over them in less time than a second launch takes
    const int sms = sm_count();
    const int64_t most = static_cast<int64_t>(sms > 0 ? sms : 148) * bwd_blocks_per_sm(bwd_threads(K, vec));
    // A row more for a block costs about 0.65 us; a block's share of dweight, written and added up, 1.3 us
    // per MB; the square root weighs the two. Measured (us) with 1, 2, 3, 4 rows a block: 1000 x 1024 bf16 9.3,
    // 8.1, 7.4, 7.9; 600 x 2048 10.5, 8.7, 8.0, 8.4; 333 x 512 4.3, 4.5, 6.2, 6.9; 4000 x 256 9.2, 9.9, 8.6, 8.0.
    // Over 16 sizes (200 to 4000 rows of 256 to 8192) it takes 3 % longer than the best count, 23 % at the last.
    const int64_t each = static_cast<int64_t>(std::sqrt(8e-6 * static_cast<double>(M) * static_cast<double>(K)) + 0.1);
    const int64_t blocks = each > 1 ? (M + each - 1) / each : M;
    return static_cast<size_t>(blocks < most ? blocks : most);
  }
  const int64_t rows = strip_rows(M, K, cols);
  return static_cast<size_t>((M + rows - 1) / rows);
}

template <typename T, int SG>
cudaError_t launch_bwd(BwdArgs p, int rows, int threads, cudaStream_t st) {
  const int64_t row_bytes =
      static_cast<int64_t>(row_pitch(static_cast<uint32_t>(p.K) * sizeof(T), SG == 0)) * (p.dh ? 3 : 2);
  int64_t stages = (kRingSmem / bwd_blocks_per_sm(threads) - 2048) / row_bytes;
  if (stages > kMaxStages) stages = kMaxStages;
  if (stages >= 2 && p.M >= 2 * rows) {
    auto kern = norm_bwd_kernel<T, true, SG>;
    static std::atomic<uint64_t> smem_set{0};
    if (set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kRingSmem, smem_set,
                             "rms_norm_bwd: set shared memory") == C3CU_OK) {
      p.stages = static_cast<int>(stages);
      kern<<<rows, threads, static_cast<size_t>(stages * row_bytes), st>>>(p);
      return cudaGetLastError();
    }
  }
  norm_bwd_kernel<T, false, SG><<<rows, threads, 0, st>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_bwd_rows(const BwdArgs& p, bool vec, int rows, int threads, cudaStream_t st) {
  if (vec) return launch_bwd<T, 0>(p, rows, threads, st);
  switch (threads) {
    case 32: return launch_bwd<T, 32>(p, rows, threads, st);
    case 64: return launch_bwd<T, 64>(p, rows, threads, st);
    case 128: return launch_bwd<T, 128>(p, rows, threads, st);
    case 256: return launch_bwd<T, 256>(p, rows, threads, st);
    default: return launch_bwd<T, 512>(p, rows, threads, st);
  }
}

// Buffers of norm_bwd_wide_kernel's ring, or 0 for strips: rows of which not two fit, or too few rows for
// a block on each SM (3 x 12288 bf16: 7.8 us in strips, 14 in this kernel; 40 rows: 14.4 both).
int wide_stages(int64_t M, int64_t K, int esize, bool vec, bool dh) {
  if (K > kWideThreads * kWideElems || M < sm_count()) return 0;
  const int64_t stages = (kRingSmem - 2048) / (row_pitch(static_cast<uint32_t>(K * esize), vec) * (dh ? 3 : 2));
  return stages < 2 ? 0 : static_cast<int>(stages < kMaxStages ? stages : kMaxStages);
}

template <typename T, int SG>
cudaError_t launch_bwd_wide(BwdArgs p, int blocks, int stages, cudaStream_t st) {
  auto kern = norm_bwd_wide_kernel<T, SG>;
  static std::atomic<uint64_t> smem_set{0};
  if (set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kRingSmem, smem_set,
                           "rms_norm_bwd: set shared memory") != C3CU_OK)
    return cudaErrorInvalidValue;
  p.stages = stages;
  kern<<<blocks, kWideThreads,
         static_cast<size_t>(stages) * row_pitch(static_cast<uint32_t>(p.K) * sizeof(T), SG == 0) * (p.dh ? 3 : 2), st>>>(p);
  return cudaGetLastError();
}

template <typename T, int SG>
cudaError_t launch_bwd_strips(BwdArgs p, float* dots, int rows, cudaStream_t st) {
  constexpr int kCols = kStripThreads * Runs<T, SG>::V;
  norm_bwd_dot_kernel<T, SG ? 512 : 0><<<p.M, 512, 0, st>>>(p, dots);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  return launch_next(norm_bwd_strip_kernel<T, SG>, dim3((p.K + kCols - 1) / kCols, rows), dim3(kStripThreads), 0, st, p,
                     static_cast<const float*>(dots), strip_rows(p.M, p.K, kCols));
}

template <typename T>
int bwd(BwdArgs p, bool vec, float* ws, cudaStream_t st) {
  const int cols = kStripThreads * (vec ? Runs<T, 0>::V : 8);
  int rows = static_cast<int>(bwd_partial_rows(p.M, p.K, vec, cols));
  const int stages = p.K > kBwdMaxK ? wide_stages(p.M, p.K, sizeof(T), vec, p.dh != nullptr) : 0;
  cudaError_t err;
  if (p.K <= kBwdMaxK) {
    p.partial = ws;
    err = launch_bwd_rows<T>(p, vec, rows, bwd_threads(p.K, vec), st);
  } else if (stages > 0) {
    rows = sm_count();  // a block on each
    p.partial = ws;
    err = vec ? launch_bwd_wide<T, 0>(p, rows, stages, st) : launch_bwd_wide<T, kWideThreads>(p, rows, stages, st);
  } else {
    p.partial = ws + p.M;
    err = vec ? launch_bwd_strips<T, 0>(p, ws, rows, st) : launch_bwd_strips<T, kStripThreads>(p, ws, rows, st);
  }
  int rc = cuda_status(err, "rms_norm_bwd: launch");
  if (rc != C3CU_OK || rows <= 1) return rc;
  err = launch_next(sum_partials_kernel, dim3((p.K + 31) / 32), dim3(1024), 0, st, static_cast<const float*>(p.partial),
                    p.dweight, rows, p.K);
  return cuda_status(err, "rms_norm_bwd: launch");
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
      if (K <= quant::kBwdMaxK) break;  // only strips depend on v
    }
  }
  if (K > quant::kBwdMaxK && M >= sm_count() && static_cast<size_t>(sm_count()) > rows) rows = sm_count();
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
