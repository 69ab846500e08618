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
  auto kern = ckpt_narrow::dw_narrow_kernel<32, false>;
  constexpr int kSmem = static_cast<int>(ckpt_narrow::Ring<32, false>::kSmem);
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

// The calling thread's choice of form (c3cu_set_int8_form): -1 none, 0 the persistent kernel, else tiles
// of that many rows, split over clusters of g_form_split.
thread_local int g_form_tile = -1, g_form_split = 1;
thread_local bool g_form_ready = false;

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
  const int64_t kb = (K + igemm::narrow::BK - 1) / igemm::narrow::BK;
  const auto tiled = [kb](int T, int split) {
    const int64_t per = (kb + split - 1) / split;
    int stages = static_cast<int>(igemm::narrow::kMaxRing / igemm::narrow::stage_bytes(T));
    if (stages > igemm::narrow::kMaxStages) stages = igemm::narrow::kMaxStages;
    if (stages > per) stages = static_cast<int>(per);
    return ForwardPlan{T, split, static_cast<int>(per), stages};
  };
  if (g_form_tile >= 0) return g_form_tile == 0 ? best : tiled(g_form_tile, g_form_split);
  if (gemm_max_ctas() > 0) return best;  // the persistent kernel keeps to the caller's CTAs
  double least = 2.5 + waves(pairs, sms / 2) * (4.0 + 0.27 * static_cast<double>(kb_pair));
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
        best = tiled(kind.T, split);
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
// cores. Measured (us in a graph, igemv / the best narrow form): one token, 4096 x 4096 5.0 / 7.4, 1024 x
// 1024 2.0 / 4.4, 12288 x 12288 25.5 / 27.9; two, 12288 x 4096 11.1 / 11.8, 16384 x 16384 44.6 / 45.7; four,
// 4096 x 4096 6.3 / 7.5, 12288 x 4096 16 / 11.8.
bool use_igemv(int64_t M, int64_t N, int64_t K) {
  if (g_form_tile >= 0) return false;
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
// CTAs, or in large ones: the operands' layout in the workspace and the tiles' plan.
struct DwRun {
  int T, split, kb_per_cta;
  bool ready;  // the operands are laid out in the workspace first (always for large tiles)
  int clusters;
  ckpt::Plan plan;
  ckpt::Prep prep;                           // sizes only
  size_t top_at, back_at, z_at, x_at, bytes;  // the workspace's parts; partial sums first
};

int dw_clusters(int* clusters) {
  auto kern = ckpt::dw_kernel;
  static std::atomic<uint64_t> smem_set{0};
  int rc = C3CU_OK;
  if (sm_count() > 0)  // before the occupancy query, which depends on it
    rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), ckpt::SMEM_BYTES, smem_set,
                              "gemm_dw_int8: set max dynamic shared memory");
  *clusters = pair_clusters(kern, ckpt::SMEM_BYTES, ckpt::kThreads);
  return rc;
}

// Up to this many rows dZ is one band, whose columns' maxima operands_kernel finds by itself: its blocks read
// their rows twice in less time than a launch takes (us in a graph, one band / two kernels: 128 x 4096 x 4096 14.7
// / 16.6, 300 x 12288 x 1024 17.5 / 19.1, 576 x 2176 x 4822 23.2 / 23.7, 640 x 2560 x 2048 17.4 / 16.6).
constexpr int64_t kOneBand = 576;

int dw_run(int64_t M, int64_t N, int64_t K, DwRun* r) {
  const int64_t tiles = ((N + ckpt::TM - 1) / ckpt::TM) * ((K + ckpt::TN - 1) / ckpt::TN);
  if (tiles > (1 << 24)) {
    set_error("gemm_dw_int8: dW is too large (N %lld, K %lld)", (long long)N, (long long)K);
    return C3CU_ERR_INVALID;
  }
  const int blocks = static_cast<int>((M + ckpt::BK - 1) / ckpt::BK);
  const int rc = dw_clusters(&r->clusters);
  if (rc != C3CU_OK) return rc;
  r->plan = ckpt::make_plan(static_cast<int>(tiles), r->clusters, blocks);
  // The fastest form by a model of all, fitted to B200 measurements (us in a graph; blocks: K blocks of 64
  // rows of X that a CTA or pair goes through):
  //   large            6.0 + waves * 2.2 + blocks 0.34 + cut tiles 2.1 + 0.107 pieces + prep
  //   small, ready     3.8 + waves (blocks c(T) + e(T)) + prep, the operands' bytes: through L2, or HBM,
  //                    less 1.0 for a launch that is not made (kOneBand)
  //   small, converted 1.2 + waves (blocks c(T) + e(T)), e for a split tile 3.2 + 0.026 T
  // Over 120 random sizes that it was not fitted to its choice takes 0.5 % longer than the fastest form on
  // average, 18 % at worst. Measured, large /
  // ready / converted: 256 x 784 over 128 rows 8.8 / 7.3 / 4.6, 1024 x 1024 over 2048 20.0 / 14.7 / 18.5,
  // 512 x 512 over 4096 18.6 / 14.6 / 15.9, 2176 x 4822 over 576 24 / 39 / 50.
  r->T = 0;
  r->ready = true;
  if (g_form_tile > 0) {
    if (g_form_tile < 32 || g_form_tile > 128) {
      set_error("gemm_dw_int8: no tiles of %d rows", g_form_tile);
      return C3CU_ERR_INVALID;
    }
    r->T = g_form_tile;
    r->split = g_form_split;
    r->kb_per_cta = (blocks + g_form_split - 1) / g_form_split;
    r->ready = g_form_ready;
  } else if (g_form_tile < 0 && gemm_max_ctas() == 0) {  // a cap: the persistent kernel keeps to it
    const double rounds = r->plan.rest > 0
                              ? static_cast<double>(r->plan.whole / r->clusters) * blocks + r->plan.kb_per_piece
                              : static_cast<double>((tiles + r->clusters - 1) / r->clusters) * blocks;
    const double turns = static_cast<double>((tiles + r->clusters - 1) / r->clusters);
    const double bytes = static_cast<double>(M) * (6. * static_cast<double>(N) + 3. * static_cast<double>(K));
    const double prep = bytes / 7.07e6 + (bytes > 42e6 ? (bytes - 42e6) / 12.9e6 : 0.) - (M <= kOneBand ? 1.0 : 0.);
    double least = 6.0 + 2.2 * turns + 0.34 * rounds + (r->plan.rest > 0 ? 2.1 + 0.107 * r->plan.rest * r->plan.pieces : 0.) + prep;
    constexpr struct {
      int T;
      double c, e;
    } kinds[2][3] = {{{32, 0.38, 2.5}, {64, 0.515, 3.05}, {128, 0.655, 4.0}},
                     {{32, 0.28, 2.3}, {64, 0.235, 2.6}, {128, 0.335, 3.85}}};
    const int64_t k_tiles = (K + ckpt_narrow::COLS - 1) / ckpt_narrow::COLS;
    const AtOnce at_once = clusters_at_once();
    for (int ready = 0; ready < 2; ++ready) {
      for (const auto& kind : kinds[ready]) {
        if (kind.T > 32 && kind.T >= 2 * N) break;  // half of it would do
        const int64_t small = k_tiles * ((N + kind.T - 1) / kind.T);
        for (int split = 1; split <= ckpt_narrow::kMaxCluster && split <= blocks; split *= 2) {
          const int per = (blocks + split - 1) / split;
          const double e = split == 1 ? kind.e : (ready ? 3.4 : 3.2) + 0.026 * kind.T;
          const double t = (ready ? 3.8 + prep : 1.2) +
                           static_cast<double>((small + at_once(split) - 1) / at_once(split)) * (per * kind.c + e);
          if (t < least) {
            least = t;
            r->T = kind.T;
            r->split = split;
            r->kb_per_cta = per;
            r->ready = ready == 1;
          }
        }
      }
    }
  }
  r->bytes = 0;
  if (!r->ready) return C3CU_OK;
  ckpt::Prep& p = r->prep;
  p = ckpt::Prep{};
  p.M = static_cast<int32_t>(M);
  p.N = static_cast<int32_t>(N);
  p.K = static_cast<int32_t>(K);
  p.tiles = static_cast<int32_t>((N + 63) / 64);
  // as many items as blocks that run at once, four an SM, so that each streams its rows without a restart
  int64_t bands = static_cast<int64_t>(sm_count() > 0 ? sm_count() : 148) * 4 / p.tiles;
  bands = bands < 1 ? 1 : bands > ckpt::kMaxBands ? ckpt::kMaxBands : bands;
  int64_t rows = (M + bands - 1) / bands;
  rows = (rows + ckpt::kPrepRows - 1) / ckpt::kPrepRows * ckpt::kPrepRows;
  if (rows < 128) rows = 128;
  if (M <= kOneBand) rows = (M + 31) / 32 * 32;
  p.band_rows = static_cast<int32_t>(rows);
  p.bands = static_cast<int32_t>((M + rows - 1) / rows);
  p.ldz = (N + 7) / 8 * 8;
  p.ldx16 = (K + 7) / 8 * 8;
  const auto part = [r](size_t bytes) {  // parts start on 256 bytes
    const size_t at = r->bytes;
    r->bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  part(r->T > 0 ? 0 : static_cast<size_t>(r->plan.rest) * r->plan.pieces * ckpt::TM * ckpt::TN * sizeof(float));
  r->top_at = part(static_cast<size_t>(p.bands) * p.tiles * 64 * sizeof(float));
  r->back_at = part(static_cast<size_t>(p.tiles) * 64 * sizeof(float));
  r->z_at = part(static_cast<size_t>(M) * p.ldz * sizeof(__half));
  r->x_at = part(static_cast<size_t>(M) * p.ldx16 * sizeof(__half));
  return C3CU_OK;
}

template <int T, bool READY>
int launch_dw_narrow(const CUtensorMap& tz, const CUtensorMap& tx, const ckpt_narrow::Params& p, int split,
                     cudaStream_t st) {
  auto kern = ckpt_narrow::dw_narrow_kernel<T, READY>;
  static std::atomic<uint64_t> smem_set{0};
  const int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), ckpt_narrow::Ring<T, READY>::kSmem, smem_set,
                                      "gemm_dw_int8: set max dynamic shared memory");
  if (rc != C3CU_OK) return rc;
  const int64_t grid = static_cast<int64_t>(p.k_tiles) * ((p.N + T - 1) / T) * split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(ckpt_narrow::kThreads);
  cfg.dynamicSmemBytes = ckpt_narrow::Ring<T, READY>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // READY: after operands_kernel
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = READY ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, tz, tx, p), "gemm_dw_int8: launch");
}

template <bool READY>
int launch_dw_tiles(const DwRun& r, const CUtensorMap& tz, const CUtensorMap& tx, const ckpt_narrow::Params& p,
                    cudaStream_t st) {
  switch (r.T) {
    case 32: return launch_dw_narrow<32, READY>(tz, tx, p, r.split, st);
    case 64: return launch_dw_narrow<64, READY>(tz, tx, p, r.split, st);
    default: return launch_dw_narrow<128, READY>(tz, tx, p, r.split, st);
  }
}

// The product from the operands in the workspace.
int launch_dw_ready(const DwRun& r, const ckpt::Prep& a, const ckpt::Params& p, cudaStream_t st) {
  // a block an item, or as many as the caller's cap
  const int64_t most = gemm_max_ctas() > 0 ? gemm_max_ctas() : INT32_MAX;
  const auto grid = [most](int64_t items) { return dim3(static_cast<unsigned>(items < most ? items : most)); };
  const int64_t dz_items = static_cast<int64_t>(a.tiles) * a.bands;
  const int64_t x_items = (static_cast<int64_t>(a.M) + ckpt::kWidenRows - 1) / ckpt::kWidenRows;
  int rc = C3CU_OK;
  if (a.bands > 1)
    rc = cuda_status(launch_kernel(ckpt::column_top_kernel, grid(dz_items), dim3(ckpt::kPrepThreads), 0, st, a),
                     "gemm_dw_int8: launch");
  if (rc != C3CU_OK) return rc;
  // with one band it is the call's first kernel
  rc = cuda_status(launch_serialized(a.bands > 1 || pdl_enabled(), ckpt::operands_kernel, grid(dz_items + x_items),
                                     dim3(ckpt::kPrepThreads), 0, st, a),
                   "gemm_dw_int8: launch");
  if (rc != C3CU_OK) return rc;
  CUtensorMap tz, tx;  // fp16, which TMA moves like any two bytes
  if ((rc = encode_bf16_2d_sw128(&tz, a.z16, p.M, p.N, a.ldz, 64, ckpt::BK)) != C3CU_OK) return rc;
  if ((rc = encode_bf16_2d_sw128(&tx, a.x16, p.M, p.K, a.ldx16, 64, ckpt::BK)) != C3CU_OK) return rc;
  if (r.T > 0) {
    const ckpt_narrow::Params q{p.M, p.N, p.K, p.out, p.ldo, p.back, r.kb_per_cta, (p.K + ckpt_narrow::COLS - 1) / ckpt_narrow::COLS};
    return launch_dw_tiles<true>(r, tz, tx, q, st);
  }
  const int items = ckpt::item_count(p.plan);
  const int clusters = items < r.clusters ? items : r.clusters;
  rc = cuda_status(launch_next(ckpt::dw_kernel, dim3(2 * clusters), dim3(ckpt::kThreads), ckpt::SMEM_BYTES, st, tz, tx, p),
                   "gemm_dw_int8: launch");
  if (rc != C3CU_OK || p.plan.rest == 0) return rc;
  return cuda_status(launch_next(ckpt::add_pieces_kernel, dim3(ckpt::TM / ckpt::kAddRows, p.plan.rest), dim3(ckpt::TN),
                                 0, st, p),
                     "gemm_dw_int8: launch");
}

}  // namespace
}  // namespace c3cu

extern "C" int c3cu_set_int8_form(int tile, int split, int ready) {
  using namespace c3cu;
  const auto power = [](int v, int lo, int hi) { return v >= lo && v <= hi && (v & (v - 1)) == 0; };
  if (tile > 0 ? !power(tile, 16, 256) || !power(split, 1, 8) : tile < -1) {
    set_error("set_int8_form: tile %d, split %d", tile, split);
    return C3CU_ERR_INVALID;
  }
  g_form_tile = tile;
  g_form_split = tile > 0 ? split : 1;
  g_form_ready = ready != 0;
  return C3CU_OK;
}

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
  return dw_run(M, N, K, &r) == C3CU_OK ? r.bytes : 0;
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
  // the same rule in both forms, of which one reads by TMA
  if ((rc = check_bf16_rows(dZ, N, lddz)) != C3CU_OK) return rc;
  if ((rc = check_int8_rows(X, K, ldx)) != C3CU_OK) return rc;
  DwRun r;
  if ((rc = dw_run(M, N, K, &r)) != C3CU_OK) return rc;
  if (r.bytes > 0 && (!workspace || workspace_bytes < r.bytes || !aligned16(workspace))) {
    set_error("gemm_dw_int8: workspace of %zu bytes (16-byte aligned), %zu needed", workspace ? workspace_bytes : 0, r.bytes);
    return C3CU_ERR_WORKSPACE;
  }
  if (!r.ready) {
    CUtensorMap tz, tx;
    if ((rc = encode_bf16_2d_sw128(&tz, dZ, M, N, lddz, 64, ckpt::BK)) != C3CU_OK) return rc;
    if ((rc = encode_int8_2d(&tx, X, M, K, ldx, ckpt_narrow::COLS, ckpt::BK, false)) != C3CU_OK) return rc;
    const ckpt_narrow::Params q{static_cast<int32_t>(M), static_cast<int32_t>(N), static_cast<int32_t>(K),
                                static_cast<__nv_bfloat16*>(dW), lddw, x_scale, r.kb_per_cta,
                                static_cast<int32_t>((K + ckpt_narrow::COLS - 1) / ckpt_narrow::COLS)};
    return launch_dw_tiles<false>(r, tz, tx, q, st);
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ckpt::Prep a = r.prep;
  a.dz = static_cast<const __nv_bfloat16*>(dZ);
  a.lddz = lddz;
  a.q = X;
  a.ldq = ldx;
  a.scale = x_scale;
  a.top = reinterpret_cast<float*>(ws + r.top_at);
  a.back = reinterpret_cast<float*>(ws + r.back_at);
  a.z16 = reinterpret_cast<__half*>(ws + r.z_at);
  a.x16 = reinterpret_cast<__half*>(ws + r.x_at);
  ckpt::Params p{};
  p.M = a.M;
  p.N = a.N;
  p.K = a.K;
  p.out = static_cast<__nv_bfloat16*>(dW);
  p.ldo = lddw;
  p.back = a.back;
  p.partial = reinterpret_cast<float*>(ws);
  p.plan = r.plan;
  return launch_dw_ready(r, a, p, st);
}
