// C-ABI entry points of the int8 GEMMs (include/c3cu.h): the Linear forward on int8 rows with
// scales (igemm.cuh) and the weight gradient from an 8-bit checkpoint (gemm_ckpt.cuh).
#include <atomic>
#include <cstdlib>

#include "gemm_ckpt.cuh"
#include "host_util.h"
#include "igemm.cuh"

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
  int rc = encode_int8_2d(&tx, o.x, p.M, p.K, o.ldx, igemm::pair::BK, gemm2::HM, true);
  if (rc == C3CU_OK) rc = encode_int8_2d(&tw, o.w, p.N, p.K, o.ldw, igemm::pair::BK, gemm2::HN, true);
  if (rc != C3CU_OK) return rc;
  auto kern = igemm::igemm_pair_kernel<F32, RELU>;
  static std::atomic<uint64_t> smem_set{0};
  rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), gemm2::SMEM_BYTES, smem_set,
                            "linear_int8: set max dynamic shared memory");
  if (rc != C3CU_OK) return rc;
  const int64_t tiles = static_cast<int64_t>((p.M + gemm2::TM - 1) / gemm2::TM) * ((p.N + gemm2::TN - 1) / gemm2::TN);
  int clusters = pair_clusters(kern, gemm2::SMEM_BYTES, gemm2::kThreads);
  if (tiles < clusters) clusters = static_cast<int>(tiles);
  return cuda_status(launch_kernel(kern, dim3(2 * clusters), dim3(gemm2::kThreads), gemm2::SMEM_BYTES, st, tx, tw, p),
                     "linear_int8: launch");
}

struct NarrowPlan {
  int T, split, kb_per_cta, stages;
};

template <int T, bool F32, bool RELU>
int launch_igemm_narrow(const Operands& o, igemm::Params p, const NarrowPlan& plan, cudaStream_t st) {
  CUtensorMap tx, tw;
  int rc = encode_int8_2d(&tw, o.w, p.N, p.K, o.ldw, igemm::narrow::BK, igemm::narrow::BN, true);
  if (rc == C3CU_OK) rc = encode_int8_2d(&tx, o.x, p.M, p.K, o.ldx, igemm::narrow::BK, T, true);
  if (rc != C3CU_OK) return rc;
  auto kern = igemm::igemm_narrow_kernel<T, F32, RELU>;
  static std::atomic<uint64_t> smem_set{0};
  rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), 227 * 1024, smem_set,
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

template <bool F32, bool RELU>
int dispatch_igemm(const Operands& o, const igemm::Params& p, cudaStream_t st) {
  const int T = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : p.M <= 128 ? 128 : 256;
  if (p.M > 256) return launch_igemm_pair<F32, RELU>(o, p, st);
  NarrowPlan plan;
  plan.T = T;
  const int kb = (p.K + 127) / 128;
  const int64_t tiles = static_cast<int64_t>((p.N + 127) / 128) * ((p.M + T - 1) / T);
  int split = 1;
  while (split < igemm::narrow::kMaxCluster && split * 2 <= kb && tiles * split * 2 <= sm_count()) split *= 2;
  plan.split = split;
  plan.kb_per_cta = (kb + split - 1) / split;
  int stages = static_cast<int>(igemm::narrow::kMaxRing / igemm::narrow::stage_bytes(T));
  if (stages > igemm::narrow::kMaxStages) stages = igemm::narrow::kMaxStages;
  plan.stages = plan.kb_per_cta < stages ? plan.kb_per_cta : stages;
  switch (T) {
    case 16: return launch_igemm_narrow<16, F32, RELU>(o, p, plan, st);
    case 32: return launch_igemm_narrow<32, F32, RELU>(o, p, plan, st);
    case 64: return launch_igemm_narrow<64, F32, RELU>(o, p, plan, st);
    case 128: return launch_igemm_narrow<128, F32, RELU>(o, p, plan, st);
    default: return launch_igemm_narrow<256, F32, RELU>(o, p, plan, st);
  }
}

int check_gemm_sizes(const char* what, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX - 256) {
    set_error("%s: sizes out of range M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
    return C3CU_ERR_INVALID;
  }
  return C3CU_OK;
}

// How a weight gradient runs: X widened in the kernel (raw) or once into the workspace, the tiles'
// plan, and the workspace's parts (partial sums first, then the widened X).
struct DwRun {
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
  const char* e = getenv("DEV_RAW");
  r->raw = e && e[0] == '1';
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
  int rc = cuda_status(launch_kernel(ckpt::dw_kernel<RAW>, dim3(2 * clusters), dim3(ckpt::Ring<RAW>::kThreads),
                                     ckpt::Ring<RAW>::kSmem, st, ta, tx, p),
                       "gemm_dw_int8: launch");
  if (rc != C3CU_OK || p.plan.rest == 0) return rc;
  ckpt::add_pieces_kernel<<<dim3(64, p.plan.rest), 256, 0, st>>>(p);
  return cuda_status(cudaGetLastError(), "gemm_dw_int8: launch");
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
  p.vec_ok = aligned16(Y) && (M == 1 || ldy * e % 16 == 0) && aligned16(w_scale) && (!bias || aligned16(bias));
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
  p.vec_ok = aligned16(dW) && (N == 1 || lddw % 8 == 0);
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
  if (r.raw) return launch_dw<true>(ta, tx, p, r.clusters, st);
  __nv_bfloat16* wide = reinterpret_cast<__nv_bfloat16*>(static_cast<uint8_t*>(workspace) + r.partial_bytes);
  const int64_t units = M * ((r.wide_ld + 15) / 16);
  const int64_t want = (units + 255) / 256, most = static_cast<int64_t>(sm_count()) * 8;
  ckpt::widen_kernel<<<static_cast<unsigned>(want < most ? want : most), 256, 0, st>>>(
      X, ldx, x_scale, wide, r.wide_ld, static_cast<int>(M), static_cast<int>(K));
  if ((rc = cuda_status(cudaGetLastError(), "gemm_dw_int8: launch")) != C3CU_OK) return rc;
  if ((rc = encode_bf16_2d_sw128(&tx, wide, M, K, r.wide_ld, 64, ckpt::BK)) != C3CU_OK) return rc;
  return launch_dw<false>(ta, tx, p, r.clusters, st);
}
