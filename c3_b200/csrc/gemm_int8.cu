// C-ABI entry points of the int8 GEMMs (include/c3cu.h): the Linear forward on int8 rows with
// scales (igemm.cuh, igemv.cuh) and the weight gradient from an 8-bit checkpoint (gemm_ckpt.cuh).
#include <atomic>

#include "gemm_ckpt.cuh"
#include "gemm_ckpt_narrow.cuh"
#include "host_util.h"
#include "igemm.cuh"
#include "igemv.cuh"

C3CU_FAULT_ACCESSORS(int8)

namespace c3cu {
namespace {

template <class Kern>
int pair_clusters(Kern kern, uint32_t smem_bytes, int threads) {
  int clusters = max_pair_clusters(kern, smem_bytes, threads);
  if (clusters <= 0) clusters = sm_count() / 2;
  if (clusters <= 0) clusters = 74;
  const int cap = gemm_max_ctas();
  if (cap > 0 && cap / 2 < clusters) clusters = cap / 2 > 0 ? cap / 2 : 1;
  return clusters;
}

struct Operands {
  const int8_t *x, *w;
  int64_t ldx, ldw;
};

template <bool F32, bool RELU>
int launch_igemm_pair(const Operands& o, const igemm::Params& p, cudaStream_t st) {
  CUtensorMap tx, tw;
  int rc = encode_int8_2d(&tw, o.w, p.N, p.K, o.ldw, igemm::pair::BK, gemm2::HM, true);
  if (rc == C3CU_OK) rc = encode_int8_2d(&tx, o.x, p.M, p.K, o.ldx, igemm::pair::BK, gemm2::HN, true);
  if (rc != C3CU_OK) return rc;
  auto kern = igemm::igemm_pair_kernel<F32, RELU>;
  static std::atomic<uint64_t> smem_set{0};
  rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), gemm2::SMEM_BYTES, smem_set,
                            "linear_int8: set max dynamic shared memory");
  if (rc != C3CU_OK) return rc;
  const int64_t tiles = static_cast<int64_t>((p.N + gemm2::TM - 1) / gemm2::TM) * ((p.M + gemm2::TN - 1) / gemm2::TN);
  int clusters = pair_clusters(kern, gemm2::SMEM_BYTES, igemm::pair::kThreads);
  if (tiles < clusters) clusters = static_cast<int>(tiles);
  return cuda_status(launch_kernel(kern, dim3(2 * clusters), dim3(igemm::pair::kThreads), gemm2::SMEM_BYTES, st, tw, tx, p),
                     "linear_int8: launch");
}

// Clusters of 1, 2, 4 and 8 CTAs of the small-tile kernels that run at once. Each such CTA takes an SM
// for itself, and a cluster stays within one group of SMs, which need not hold a whole number of them:
// a B200 ran 74 clusters of two, but 33 of four and 15 of eight.
struct AtOnce {
  int of[4];
  int operator()(int split) const { return of[split >= 8 ? 3 : split >= 4 ? 2 : split - 1]; }
};

int query_clusters(int split) {
  auto kern = ckpt_narrow::dw_narrow_kernel<32>;
  constexpr int kSmem = static_cast<int>(ckpt_narrow::Ring<32>::kSmem);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(split) * 64);
  cfg.blockDim = dim3(ckpt_narrow::kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(split);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n;
}

AtOnce clusters_at_once() {  // asked once per device
  static std::atomic<int> cached[64][4] = {};
  AtOnce r;
  const int sms = sm_count() > 0 ? sm_count() : 148;
  int dev = 0;
  const bool known = sm_count() > 0 && cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
  for (int i = 0; i < 4; ++i) {
    const int split = 1 << i;
    r.of[i] = split == 1 || !known ? 0 : cached[dev][i].load(std::memory_order_relaxed);
    if (r.of[i] > 0) continue;
    const int n = split == 1 || !known ? 0 : query_clusters(split);
    r.of[i] = n > 0 ? n : sms / split > 0 ? sms / split : 1;
    if (n > 0) cached[dev][i].store(n, std::memory_order_relaxed);
  }
  return r;
}

// How a forward runs: T = 0 for the pair kernel, else tiles of T tokens, each split along K over a
// cluster of `split` CTAs.
struct ForwardPlan {
  int T, split, kb_per_cta, stages;
};

// The faster kernel by a model of both, fitted to B200 measurements (us; kb = K blocks of a CTA):
//   narrow  3.2 + waves (kb c(T) + e(T)), e being the epilogue, or for a split tile the exchange of
//           partial sums 1.2 + 0.028 tokens
//   pair    2.5 + waves (4.0 + 0.27 kb)
// Over 196 random sizes its choice takes 1.4 % longer than the fastest form on average.
// Measured (us), 4096 channels x K 4096: 8 tokens 5.8 (T 16, split 4) against 13.4 (pair), 64 tokens
// 7.8 (T 64, split 4) / 13.6, 512 tokens 12.5 (T 128) / 16.8, 1024 tokens 19.0 (T 256) / 17.9; 12288
// channels x K 1024, 2048 tokens 54 (T 256) / 34.
ForwardPlan plan_forward(int64_t M, int64_t N, int64_t K) {
  constexpr struct {
    int T;
    double c, e;
  } kinds[] = {{16, 0.21, 0.6}, {32, 0.22, 0.8}, {64, 0.23, 1.3}, {128, 0.27, 2.1}, {256, 0.40, 4.8}};
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const auto waves = [](int64_t work, int64_t at_once) { return static_cast<double>((work + at_once - 1) / at_once); };
  const int64_t kb_pair = (K + igemm::pair::BK - 1) / igemm::pair::BK;
  const int64_t pairs = ((N + gemm2::TM - 1) / gemm2::TM) * ((M + gemm2::TN - 1) / gemm2::TN);
  ForwardPlan best{0, 1, 0, 0};
  if (gemm_max_ctas() > 0) return best;  // the persistent kernel keeps to the caller's CTAs
  double least = 2.5 + waves(pairs, sms / 2) * (4.0 + 0.27 * static_cast<double>(kb_pair));
  const int64_t kb = (K + igemm::narrow::BK - 1) / igemm::narrow::BK;
  const AtOnce at_once = clusters_at_once();
  const int64_t n_tiles = (N + igemm::narrow::BN - 1) / igemm::narrow::BN;
  for (const auto& kind : kinds) {
    if (kind.T > 16 && kind.T >= 2 * M) break;  // half of it would do
    const int64_t tiles = n_tiles * ((M + kind.T - 1) / kind.T);
    for (int split = 1; split <= igemm::narrow::kMaxCluster && split <= kb; split *= 2) {
      const int64_t per = (kb + split - 1) / split;
      const double exchange = 1.2 + 0.028 * static_cast<double>(M < kind.T ? M : kind.T);
      const double tile = static_cast<double>(per) * kind.c + (split > 1 ? exchange : kind.e);
      const double t = 3.2 + waves(tiles, at_once(split)) * tile;
      if (t < least) {
        least = t;
        int stages = static_cast<int>(igemm::narrow::kMaxRing / igemm::narrow::stage_bytes(kind.T));
        if (stages > igemm::narrow::kMaxStages) stages = igemm::narrow::kMaxStages;
        if (stages > per) stages = static_cast<int>(per);
        best = {kind.T, split, static_cast<int>(per), stages};
      }
    }
  }
  return best;
}

template <int T, bool F32, bool RELU>
int launch_igemm_narrow(const Operands& o, igemm::Params p, const ForwardPlan& plan, cudaStream_t st) {
  CUtensorMap tx, tw;
  int rc = encode_int8_2d(&tw, o.w, p.N, p.K, o.ldw, igemm::narrow::BK, igemm::narrow::BN, true);
  if (rc == C3CU_OK) rc = encode_int8_2d(&tx, o.x, p.M, p.K, o.ldx, igemm::narrow::BK, T, true);
  if (rc != C3CU_OK) return rc;
  auto kern = igemm::igemm_narrow_kernel<T, F32, RELU>;
  static std::atomic<uint64_t> smem_set{0};
  rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), igemm::narrow::kMaxSmem, smem_set,
                            "linear_int8: set max dynamic shared memory");
  if (rc != C3CU_OK) return rc;
  p.n_tiles = (p.N + igemm::narrow::BN - 1) / igemm::narrow::BN;
  p.kb_per_cta = plan.kb_per_cta;
  p.stages = plan.stages;
  const int64_t grid = static_cast<int64_t>(p.n_tiles) * ((p.M + T - 1) / T) * plan.split;
  if (grid > INT32_MAX) {
    set_error("linear_int8: grid too large");
    return C3CU_ERR_INVALID;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(igemm::narrow::kThreads);
  cfg.dynamicSmemBytes = igemm::narrow::smem_bytes(T, plan.stages);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(plan.split);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, tw, tx, p), "linear_int8: launch");
}

// Warps per block of igemv_kernel. Few blocks: a warp for each 512 bytes of a row, so that all of W is
// asked for at once; many: one for each 1024, so that a warp has 16 loads in flight. Measured with one
// token (us): 512 channels x K 2048 2.3 with 4 warps, 3.2 with 1; 16 x 16384 3.2 with 16, 4.5 with 4;
// 12288 x 1024 4.8 with 1, 5.8 with 2; 12288 x 12288 25.9 with 4, 28.1 with 8.
int igemv_split(int64_t blocks, int64_t K) {
  const int sms = sm_count();
  const int most = blocks <= sms ? igemv::kMaxSplit : blocks <= 2 * sms ? 8 : 4;
  const int64_t each = igemv::kStep * (blocks <= 2 * sms ? 1 : igemv::kAhead);
  int split = 1;
  while (split < most && split * each < K) split *= 2;
  return split;
}

// Up to two tokens always, up to four while their multiplications do not outweigh a tile on the tensor
// cores. Measured (us, igemv / narrow): one token, 4096 x 4096 5.2 / 7.3, 1397 x 777 2.4 / 4.7, 12288 x
// 12288 26 / 34.5; two, 12288 x 4096 12.8 / 11.9; four, 4096 x 4096 7.1 / 7.7, 12288 x 4096 16 / 11.9.
bool use_igemv(int64_t M, int64_t N, int64_t K) {
  if (gemm_max_ctas() > 0) return false;  // the persistent kernel keeps to the caller's CTAs
  return M <= 2 || (M <= igemv::kMaxTokens && N * K <= 20'000'000);
}

template <int T, bool F32, bool RELU>
int launch_igemv(const Operands& o, const igemm::Params& p, cudaStream_t st) {
  int rc = check_int8_rows(o.w, p.K, o.ldw);
  if (rc == C3CU_OK) rc = check_int8_rows(o.x, p.K, o.ldx);
  if (rc != C3CU_OK) return rc;
  // a block writes a byte of the mask: those past N complete the rows' last words
  const int64_t channels = RELU && p.mask ? (static_cast<int64_t>(p.N) + 31) / 32 * 32 : p.N;
  const int64_t blocks = (channels + igemv::kChannels - 1) / igemv::kChannels;
  const int split = igemv_split(blocks, p.K);
  return cuda_status(launch_kernel(igemv::igemv_kernel<T, F32, RELU>, dim3(static_cast<unsigned>(blocks)),
                                   dim3(32 * split), 0, st, o.x, o.ldx, o.w, o.ldw, p),
                     "linear_int8: launch");
}

template <bool F32, bool RELU>
int dispatch_igemm(const Operands& o, const igemm::Params& p, cudaStream_t st) {
  if (use_igemv(p.M, p.N, p.K)) {
    if (p.M == 1) return launch_igemv<1, F32, RELU>(o, p, st);
    if (p.M == 2) return launch_igemv<2, F32, RELU>(o, p, st);
    return launch_igemv<4, F32, RELU>(o, p, st);
  }
  const ForwardPlan plan = plan_forward(p.M, p.N, p.K);
  switch (plan.T) {
    case 16: return launch_igemm_narrow<16, F32, RELU>(o, p, plan, st);
    case 32: return launch_igemm_narrow<32, F32, RELU>(o, p, plan, st);
    case 64: return launch_igemm_narrow<64, F32, RELU>(o, p, plan, st);
    case 128: return launch_igemm_narrow<128, F32, RELU>(o, p, plan, st);
    case 256: return launch_igemm_narrow<256, F32, RELU>(o, p, plan, st);
    default: return launch_igemm_pair<F32, RELU>(o, p, st);
  }
}

int check_gemm_sizes(const char* what, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX - 256) {
    set_error("%s: sizes out of range M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
    return C3CU_ERR_INVALID;
  }
  return C3CU_OK;
}

// How a weight gradient runs: in small tiles (T > 0) of T rows, each split over a cluster of `split`
// CTAs, or in large ones: X widened in the kernel (raw) or once into the workspace, the tiles' plan,
// and the workspace's parts (partial sums first, then the widened X).
struct DwRun {
  int T, split, kb_per_cta;
  bool raw;
  int clusters;
  ckpt::Plan plan;
  size_t partial_bytes, wide_bytes;
  int64_t wide_ld;
};

template <bool RAW>
int dw_clusters(int* clusters) {
  auto kern = ckpt::dw_kernel<RAW>;
  static std::atomic<uint64_t> smem_set{0};
  int rc = C3CU_OK;
  if (sm_count() > 0)  // before the occupancy query, which depends on it
    rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), ckpt::Ring<RAW>::kSmem, smem_set,
                              "gemm_dw_int8: set max dynamic shared memory");
  *clusters = pair_clusters(kern, ckpt::Ring<RAW>::kSmem, ckpt::Ring<RAW>::kThreads);
  return rc;
}

int dw_run(int64_t M, int64_t N, int64_t K, DwRun* r) {
  const int64_t tiles = ((N + ckpt::TM - 1) / ckpt::TM) * ((K + ckpt::TN - 1) / ckpt::TN);
  const int blocks = static_cast<int>((M + ckpt::BK - 1) / ckpt::BK);
  // Widening X in the kernel slows each K block by about 0.2 us (0.6 instead of 0.4); widening it first
  // costs a launch, about 2.5 us, and three bytes per element of X at 6 TB/s.
  dw_clusters<true>(&r->clusters);
  r->plan = ckpt::make_plan(static_cast<int>(tiles), r->clusters, blocks);
  const double rounds = static_cast<double>(r->plan.whole / r->clusters) * blocks +
                        (r->plan.rest > 0 ? r->plan.kb_per_piece : 0);
  const double whole_only = r->plan.rest > 0 ? rounds : static_cast<double>((tiles + r->clusters - 1) / r->clusters) * blocks;
  const double widening = 3. * static_cast<double>(M) * static_cast<double>(K) / 6e6;
  r->raw = 0.2 * whole_only < 2.5 + widening;
  // The faster kernel by a model of both, fitted to B200 measurements (us; K blocks of 64 rows of X):
  //   large  3.3 + waves * 2.6 + blocks (0.43 RAW, 0.36 else) + cut tiles 2.8 + 0.09 pieces + widening
  //   small  1.3 + waves (blocks c(T) + e(T)), e for a split tile 3.5 + 0.021 T
  // Over 57 random sizes it misses the fastest form by 0.8 % on average, large tiles alone by 29 %.
  // Measured, small / large: 256 x 784 over 128 rows 4.1 / 6.5, 32 x 25 over 2908 6.9 / 11.1, 1024 x
  // 1024 over 2048 13.8 / 15.9, 2176 x 4822 over 576 37 / 21.
  r->T = 0;
  if (gemm_max_ctas() == 0) {  // else the persistent kernel keeps to the caller's CTAs
    const double turns = static_cast<double>((tiles + r->clusters - 1) / r->clusters);
    double least = 3.3 + 2.6 * turns + (r->raw ? 0.43 : 0.36) * whole_only +
                   (r->plan.rest > 0 ? 2.8 + 0.09 * r->plan.rest * r->plan.pieces : 0.) + (r->raw ? 0. : 1. + widening);
    constexpr struct {
      int T;
      double c, e;
    } kinds[] = {{32, 0.37, 2.6}, {64, 0.40, 2.9}, {128, 0.44, 3.8}};
    const int64_t k_tiles = (K + ckpt_narrow::COLS - 1) / ckpt_narrow::COLS;
    const AtOnce at_once = clusters_at_once();
    for (const auto& kind : kinds) {
      if (kind.T > 32 && kind.T >= 2 * N) break;  // half of it would do
      const int64_t small = k_tiles * ((N + kind.T - 1) / kind.T);
      for (int split = 1; split <= ckpt_narrow::kMaxCluster && split <= blocks; split *= 2) {
        const int per = (blocks + split - 1) / split;
        const double t = 1.3 + static_cast<double>((small + at_once(split) - 1) / at_once(split)) *
                                   (per * kind.c + (split > 1 ? 3.5 + 0.021 * kind.T : kind.e));
        if (t < least) {
          least = t;
          r->T = kind.T;
          r->split = split;
          r->kb_per_cta = per;
        }
      }
    }
  }
  if (r->T > 0) {
    r->partial_bytes = r->wide_bytes = 0;
    return C3CU_OK;
  }
  const int rc = r->raw ? dw_clusters<true>(&r->clusters) : dw_clusters<false>(&r->clusters);
  r->plan = ckpt::make_plan(static_cast<int>(tiles), r->clusters, blocks);
  r->partial_bytes = static_cast<size_t>(r->plan.rest) * r->plan.pieces * ckpt::TM * ckpt::TN * sizeof(float);
  r->wide_ld = (K + 7) / 8 * 8;
  r->wide_bytes = r->raw ? 0 : static_cast<size_t>(M) * r->wide_ld * 2;
  return rc;
}

template <bool RAW>
int launch_dw(const CUtensorMap& ta, const CUtensorMap& tx, const ckpt::Params& p, int clusters, cudaStream_t st) {
  const int items = ckpt::item_count(p.plan);
  if (items < clusters) clusters = items;
  // not RAW: the kernel that widens X is before it
  int rc = cuda_status(launch_serialized(!RAW || pdl_enabled(), ckpt::dw_kernel<RAW>, dim3(2 * clusters),
                                         dim3(ckpt::Ring<RAW>::kThreads), ckpt::Ring<RAW>::kSmem, st, ta, tx, p),
                       "gemm_dw_int8: launch");
  if (rc != C3CU_OK || p.plan.rest == 0) return rc;
  return cuda_status(launch_next(ckpt::add_pieces_kernel, dim3(ckpt::TM / ckpt::kAddRows, p.plan.rest), dim3(ckpt::TN),
                                 0, st, p),
                     "gemm_dw_int8: launch");
}

template <int T>
int launch_dw_narrow(const CUtensorMap& tz, const CUtensorMap& tx, const ckpt_narrow::Params& p, int split,
                     cudaStream_t st) {
  auto kern = ckpt_narrow::dw_narrow_kernel<T>;
  static std::atomic<uint64_t> smem_set{0};
  const int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), ckpt_narrow::Ring<T>::kSmem, smem_set,
                            "gemm_dw_int8: set max dynamic shared memory");
  if (rc != C3CU_OK) return rc;
  const int64_t grid = static_cast<int64_t>(p.k_tiles) * ((p.N + T - 1) / T) * split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(ckpt_narrow::kThreads);
  cfg.dynamicSmemBytes = ckpt_narrow::Ring<T>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(split);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, tz, tx, p), "gemm_dw_int8: launch");
}

}  // namespace
}  // namespace c3cu

extern "C" int c3cu_linear_int8_fwd(const int8_t* X, int64_t ldx, const float* x_scale, const int8_t* W, int64_t ldw,
                                    const float* w_scale, const float* bias, void* Y, int64_t ldy, int out_dtype,
                                    int relu, uint32_t* mask, int64_t ldm, int64_t M, int64_t N, int64_t K,
                                    c3cu_stream_t stream) {
  using namespace c3cu;
  int rc = check_gemm_sizes("linear_int8", M, N, K);
  if (rc != C3CU_OK) return rc;
  if ((rc = require_sm100()) != C3CU_OK) return rc;
  if (out_dtype != C3CU_DTYPE_F32 && out_dtype != C3CU_DTYPE_BF16) {
    set_error("linear_int8: output dtype %d is neither f32 nor bf16", out_dtype);
    return C3CU_ERR_INVALID;
  }
  if (M == 0 || N == 0) return C3CU_OK;
  if (K < 1 || K > C3CU_INT8_MAX_K) {
    set_error("linear_int8: K = %lld outside [1, %d] (the int32 sums could overflow beyond)", (long long)K,
              C3CU_INT8_MAX_K);
    return C3CU_ERR_INVALID;
  }
  if (!X || !x_scale || !W || !w_scale || !Y) {
    set_error("linear_int8: null operand");
    return C3CU_ERR_INVALID;
  }
  if (mask && !relu) {
    set_error("linear_int8: a mask belongs to the ReLU output");
    return C3CU_ERR_INVALID;
  }
  if (M > 1 && (ldy < N || (mask && ldm < (N + 31) / 32))) {
    set_error("linear_int8: output row stride %lld < N %lld, or mask row stride too small", (long long)ldy, (long long)N);
    return C3CU_ERR_INVALID;
  }
  const int e = out_dtype == C3CU_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(Y) % e || reinterpret_cast<uintptr_t>(x_scale) % 4 ||
      reinterpret_cast<uintptr_t>(w_scale) % 4 || reinterpret_cast<uintptr_t>(bias) % 4 ||
      reinterpret_cast<uintptr_t>(mask) % 4) {
    set_error("linear_int8: a pointer is not aligned to its type");
    return C3CU_ERR_ALIGN;
  }
  igemm::Params p{};
  p.M = static_cast<int32_t>(M);
  p.N = static_cast<int32_t>(N);
  p.K = static_cast<int32_t>(K);
  p.out = Y;
  p.ldo = ldy;
  p.xs = x_scale;
  p.ws = w_scale;
  p.bias = bias;
  p.mask = mask;
  p.ldm = ldm;
  const Operands o{X, W, ldx, ldw};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == C3CU_DTYPE_F32)
    return relu ? dispatch_igemm<true, true>(o, p, st) : dispatch_igemm<true, false>(o, p, st);
  return relu ? dispatch_igemm<false, true>(o, p, st) : dispatch_igemm<false, false>(o, p, st);
}

extern "C" size_t c3cu_gemm_dw_int8_workspace(int64_t M, int64_t N, int64_t K) {
  using namespace c3cu;
  if (M < 1 || N < 1 || K < 1 || check_gemm_sizes("gemm_dw_int8", M, N, K) != C3CU_OK) return 0;
  DwRun r;
  dw_run(M, N, K, &r);
  return r.partial_bytes + r.wide_bytes;
}

extern "C" int c3cu_gemm_dw_int8(const void* dZ, int64_t lddz, const int8_t* X, int64_t ldx, const float* x_scale,
                                 void* dW, int64_t lddw, int64_t M, int64_t N, int64_t K, void* workspace,
                                 size_t workspace_bytes, c3cu_stream_t stream) {
  using namespace c3cu;
  int rc = check_gemm_sizes("gemm_dw_int8", M, N, K);
  if (rc != C3CU_OK) return rc;
  if ((rc = require_sm100()) != C3CU_OK) return rc;
  if (N == 0 || K == 0) return C3CU_OK;
  if (!dW || (N > 1 && lddw < K)) {
    set_error("gemm_dw_int8: dW is null or its row stride %lld is smaller than K %lld", (long long)lddw, (long long)K);
    return C3CU_ERR_INVALID;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (M == 0)  // the sum over no rows
    return cuda_status(cudaMemset2DAsync(dW, static_cast<size_t>(N > 1 ? lddw : K) * 2, 0, static_cast<size_t>(K) * 2,
                                         static_cast<size_t>(N), st),
                       "gemm_dw_int8: clear dW");
  if (!dZ || !X || !x_scale) {
    set_error("gemm_dw_int8: null operand");
    return C3CU_ERR_INVALID;
  }
  if (reinterpret_cast<uintptr_t>(dW) % 2 || reinterpret_cast<uintptr_t>(x_scale) % 4) {
    set_error("gemm_dw_int8: a pointer is not aligned to its type");
    return C3CU_ERR_ALIGN;
  }
  ckpt::Params p{};
  p.M = static_cast<int32_t>(M);
  p.N = static_cast<int32_t>(N);
  p.K = static_cast<int32_t>(K);
  p.out = static_cast<__nv_bfloat16*>(dW);
  p.ldo = lddw;
  p.scale = x_scale;
  p.partial = static_cast<float*>(workspace);
  if (((N + 255) / 256) * ((K + 255) / 256) > (1 << 24)) {
    set_error("gemm_dw_int8: dW is too large (N %lld, K %lld)", (long long)N, (long long)K);
    return C3CU_ERR_INVALID;
  }
  DwRun r;
  if ((rc = dw_run(M, N, K, &r)) != C3CU_OK) return rc;
  p.plan = r.plan;
  const size_t need = r.partial_bytes + r.wide_bytes;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
    set_error("gemm_dw_int8: workspace of %zu bytes (16-byte aligned), %zu needed", workspace ? workspace_bytes : 0, need);
    return C3CU_ERR_WORKSPACE;
  }
  CUtensorMap ta, tx;
  if ((rc = encode_bf16_2d_sw128(&ta, dZ, M, N, lddz, 64, ckpt::BK)) != C3CU_OK) return rc;
  // X's rows are checked by the same rule in both forms
  if ((rc = encode_int8_2d(&tx, X, M, K, ldx, ckpt::HN, ckpt::BK, false)) != C3CU_OK) return rc;
  if (r.T > 0) {
    const ckpt_narrow::Params q{p.M, p.N, p.K, p.out, p.ldo, p.scale, r.kb_per_cta,
                                (p.K + ckpt_narrow::COLS - 1) / ckpt_narrow::COLS};
    switch (r.T) {
      case 32: return launch_dw_narrow<32>(ta, tx, q, r.split, st);
      case 64: return launch_dw_narrow<64>(ta, tx, q, r.split, st);
      default: return launch_dw_narrow<128>(ta, tx, q, r.split, st);
    }
  }
  if (r.raw) return launch_dw<true>(ta, tx, p, r.clusters, st);
  __nv_bfloat16* wide = reinterpret_cast<__nv_bfloat16*>(static_cast<uint8_t*>(workspace) + r.partial_bytes);
  const int64_t want = (M + ckpt::kWidenWarps - 1) / ckpt::kWidenWarps, most = static_cast<int64_t>(sm_count()) * 8;
  rc = cuda_status(launch_kernel(ckpt::widen_kernel, dim3(static_cast<unsigned>(want < most ? want : most)),
                                 dim3(32 * ckpt::kWidenWarps), 0, st, X, ldx, x_scale, wide, r.wide_ld,
                                 static_cast<int>(M), static_cast<int>(K)),
                   "gemm_dw_int8: launch");
  if (rc != C3CU_OK) return rc;
  if ((rc = encode_bf16_2d_sw128(&tx, wide, M, K, r.wide_ld, 64, ckpt::BK)) != C3CU_OK) return rc;
  return launch_dw<false>(ta, tx, p, r.clusters, st);
}
