// C ABI of the vllm-exact B200 library (declarations and contracts: include/vllm_exact_b200.h).
//
// The whole library is one translation unit (this file includes the kernel headers) so that every kernel shares the
// single device error word g_ex_dev_error. Every entry point validates its arguments before launching anything,
// never allocates device memory and never synchronizes the host.
#include <cstring>
#include <mutex>
#include <string>

#include "ex_common.cuh"
#include "ex_tp_fused.cuh"
#include "ex_digitize.cuh"
#include "ex_gemm_simt.cuh"
#include "ex_gemm_tc.cuh"
#include "ex_paged_decode.cuh"
#include "ex_paged_decode_tma.cuh"
#include "ex_cache_q8.cuh"
#include "ex_paged_rows.cuh"
#include "ex_prompt_attn.cuh"
#include "ex_tree_tc.cuh"

// Split-K scratch of ex_linear_noalloc: a file-scope device array, so that entry point never allocates. Host code
// must not hand this symbol to a kernel (on the host it is only a stand-in); the device address is looked up once per
// device with cudaGetSymbolAddress.
static __device__ __align__(256) unsigned char g_ex_noalloc_scratch[EX_NOALLOC_SCRATCH_BYTES];

namespace {

thread_local std::string g_last_error;

int cuda_status(cudaError_t e) {
  if (e == cudaSuccess) return EX_OK;
  g_last_error = cudaGetErrorString(e);
  return EX_ERR_CUDA;
}

bool dtype_ok(int d) { return d == EX_DTYPE_F32 || d == EX_DTYPE_BF16 || d == EX_DTYPE_F16; }
size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

int num_sms() {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
      sms = v;
    else
      sms = 148;
  }
  return sms;
}

// ---------------------------------------------------------------------------------------------------------------
// SIMT plan: row blocks of 256 weight rows, K split so that there are about two CTAs per SM.
// ---------------------------------------------------------------------------------------------------------------
struct SimtPlan {
  int splits;
  int kchunk;
  int nblocks;
  size_t ws_bytes;
};

SimtPlan simt_plan(int64_t M, int64_t N, int64_t K, int split_k) {
  SimtPlan p;
  p.nblocks = (int)cdiv(N, ex::SIMT_THREADS);
  int s = split_k;
  if (s <= 0) {
    const int target = 2 * num_sms();
    s = (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(target, p.nblocks), K / 256));
  }
  s = (int)std::max<int64_t>(1, std::min<int64_t>(s, std::max<int64_t>(1, cdiv(K, 16))));
  p.kchunk = (int)std::max<int64_t>(16, align_up((size_t)cdiv(K, s), 16));
  p.splits = K > 0 ? (int)cdiv(K, p.kchunk) : 1;
  p.ws_bytes = p.splits > 1 ? align_up((size_t)p.nblocks * 4, 256) + (size_t)M * N * 8 : 0;
  return p;
}

template <int F, bool TRUNC, int OD, bool PARTIAL>
cudaError_t launch_simt_t(const int8_t* xh, const int8_t* xl, int64_t ldx, const int32_t* cx, const int32_t* sx,
                          const int8_t* wh, const int8_t* wl, int64_t ldw, const int32_t* cw, const int32_t* sw,
                          int M, int N, int K, const SimtPlan& p, void* out, int64_t ldo, void* ws, cudaStream_t st) {
  const bool vecw = (ldw % 16 == 0) && (reinterpret_cast<uintptr_t>(wh) % 16 == 0) &&
                    (reinterpret_cast<uintptr_t>(wl) % 16 == 0);
  int* cnt = reinterpret_cast<int*>(ws);
  long long* acc = p.splits > 1 ? reinterpret_cast<long long*>(reinterpret_cast<char*>(ws) +
                                                               align_up((size_t)p.nblocks * 4, 256))
                                 : nullptr;
  dim3 grid(p.nblocks, p.splits);
  ex::k_exact_simt<F, TRUNC, OD, PARTIAL><<<grid, ex::SIMT_THREADS, 0, st>>>(
      xh, xl, ldx, cx, sx, wh, wl, ldw, cw, sw, M, N, K, p.kchunk, vecw, out, ldo, acc, cnt);
  return cudaGetLastError();
}

template <bool PARTIAL>
cudaError_t launch_simt(int F, int trunc, int od, const int8_t* xh, const int8_t* xl, int64_t ldx, const int32_t* cx,
                        const int32_t* sx, const int8_t* wh, const int8_t* wl, int64_t ldw, const int32_t* cw,
                        const int32_t* sw, int M, int N, int K, const SimtPlan& p, void* out, int64_t ldo, void* ws,
                        cudaStream_t st) {
#define EX_SIMT_CASE(FF, TT, OO)                                                                              \
  if (F == FF && (trunc != 0) == TT && (PARTIAL || od == OO))                                                 \
    return launch_simt_t<FF, TT, OO, PARTIAL>(xh, xl, ldx, cx, sx, wh, wl, ldw, cw, sw, M, N, K, p, out, ldo, \
                                              ws, st);
  EX_SIMT_CASE(14, true, EX_DTYPE_BF16)
  EX_SIMT_CASE(14, true, EX_DTYPE_F32)
  EX_SIMT_CASE(14, true, EX_DTYPE_F16)
  EX_SIMT_CASE(14, false, EX_DTYPE_BF16)
  EX_SIMT_CASE(14, false, EX_DTYPE_F32)
  EX_SIMT_CASE(14, false, EX_DTYPE_F16)
  EX_SIMT_CASE(15, true, EX_DTYPE_BF16)
  EX_SIMT_CASE(15, true, EX_DTYPE_F32)
  EX_SIMT_CASE(15, true, EX_DTYPE_F16)
  EX_SIMT_CASE(15, false, EX_DTYPE_BF16)
  EX_SIMT_CASE(15, false, EX_DTYPE_F32)
  EX_SIMT_CASE(15, false, EX_DTYPE_F16)
#undef EX_SIMT_CASE
  return cudaErrorInvalidValue;
}

// Shared argument validation of ex_linear / ex_linear_partial_i64.
int check_linear_args(const int8_t* xh, const int8_t* xl, int64_t ldx, const int32_t* cx, const int8_t* wh,
                      const int8_t* wl, int64_t ldw, const int32_t* cw, int64_t M, int64_t N, int64_t K, int F,
                      const void* out, int64_t ldo) {
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX || N > INT32_MAX) return EX_ERR_ARG;
  if (K > ex::EX_MAX_K) return EX_ERR_UNSUPPORTED;
  if (F != 14 && F != 15) return EX_ERR_ARG;
  if (M == 0 || N == 0) return EX_OK;
  if (!out || ldo < N) return EX_ERR_ARG;
  if (K > 0 && (!xh || !xl || !wh || !wl || ldx < K || ldw < K)) return EX_ERR_ARG;
  if (F == 15 && (!cx || !cw)) return EX_ERR_ARG;
  return EX_OK;
}

// Algorithm choice for EX_ALGO_AUTO: the tcgen05 int8 kernel whenever its TMA alignment rules hold, else SIMT.
int pick_algo(int algo, const int8_t* xh, const int8_t* xl, int64_t ldx, const int8_t* wh, const int8_t* wl,
              int64_t ldw, int64_t M, int64_t N, int64_t K) {
  if (algo != EX_ALGO_AUTO) return algo;
  if (ex::tc_supported(xh, xl, ldx, wh, wl, ldw, M, N, K)) return EX_ALGO_TC_I8;
  return EX_ALGO_SIMT;
}

template <bool PARTIAL>
int linear_impl(const int8_t* xh, const int8_t* xl, int64_t ldx, const int32_t* cx, const int32_t* sx,
                const int8_t* wh, const int8_t* wl, int64_t ldw, const int32_t* cw, const int32_t* sw, int64_t M,
                int64_t N, int64_t K, int F, int trunc, void* out, int out_dtype, int64_t ldo, void* workspace,
                size_t workspace_bytes, int split_k, int algo, cudaStream_t st) {
  int rc = check_linear_args(xh, xl, ldx, cx, wh, wl, ldw, cw, M, N, K, F, out, ldo);
  if (rc != EX_OK || M == 0 || N == 0) return rc;
  if (!PARTIAL && (!sx || !sw)) return EX_ERR_ARG;
  if (!PARTIAL && !dtype_ok(out_dtype)) return EX_ERR_DTYPE;
  if (split_k < 0) return EX_ERR_ARG;
  const bool static_w = (algo & EX_LINEAR_STATIC_WEIGHTS) != 0;
  algo = pick_algo(algo & ~EX_LINEAR_STATIC_WEIGHTS, xh, xl, ldx, wh, wl, ldw, M, N, K);
  if (algo == EX_ALGO_SIMT) {
    const SimtPlan p = simt_plan(M, N, K, split_k);
    if (p.ws_bytes > 0 && (!workspace || workspace_bytes < p.ws_bytes)) return EX_ERR_WORKSPACE;
    if (p.ws_bytes > 0 && reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return EX_ERR_ALIGN;
    return cuda_status(launch_simt<PARTIAL>(F, trunc, out_dtype, xh, xl, ldx, cx, sx, wh, wl, ldw, cw, sw, (int)M,
                                            (int)N, (int)K, p, out, ldo, workspace, st));
  }
  if (algo == EX_ALGO_TC_I8) {
    if (!ex::tc_supported(xh, xl, ldx, wh, wl, ldw, M, N, K)) return EX_ERR_ALIGN;
    const ex::TcPlan p = ex::tc_plan(M, N, K, split_k, num_sms(), ex::tc_cluster_cap());
    if (p.ws_bytes > 0 && (!workspace || workspace_bytes < p.ws_bytes)) return EX_ERR_WORKSPACE;
    if (p.ws_bytes > 0 && reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return EX_ERR_ALIGN;
    cudaError_t e = ex::launch_tc<PARTIAL>(p, F, trunc, out_dtype, xh, xl, ldx, cx, sx, wh, wl, ldw, cw, sw, (int)M,
                                           (int)N, (int)K, out, ldo, workspace, static_w, st);
    if (e == cudaErrorNotSupported) return EX_ERR_UNSUPPORTED;
    return cuda_status(e);
  }
  return EX_ERR_ARG;
}

// Per-device address of g_ex_noalloc_scratch, looked up (and the array cleared) on the first call on each device.
std::mutex g_noalloc_mu;
void* g_noalloc_ptr[128] = {};

int noalloc_scratch(cudaStream_t st, void** out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  if (dev < 0 || dev >= 128) return EX_ERR_UNSUPPORTED;
  std::lock_guard<std::mutex> lock(g_noalloc_mu);
  if (!g_noalloc_ptr[dev]) {
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_ex_noalloc_scratch);
    if (e != cudaSuccess) return cuda_status(e);
    e = cudaMemsetAsync(p, 0, EX_NOALLOC_SCRATCH_BYTES, st);  // split-K slots and tickets must start at zero
    if (e != cudaSuccess) return cuda_status(e);
    g_noalloc_ptr[dev] = p;
  }
  *out = g_noalloc_ptr[dev];
  return EX_OK;
}

// Clears the scratch of every device that has used it (synchronously, each with its own device current). A call
// that stopped early on a timed-out wait can leave split-K partials and tickets behind; ex_device_error() calls this
// whenever it reports such an error, so later calls start from zero again.
int noalloc_clear_all() {
  int cur = 0;
  cudaError_t e = cudaGetDevice(&cur);
  if (e != cudaSuccess) return cuda_status(e);
  std::lock_guard<std::mutex> lock(g_noalloc_mu);
  int rc = EX_OK;
  for (int d = 0; d < 128; ++d) {
    if (!g_noalloc_ptr[d]) continue;
    if ((e = cudaSetDevice(d)) == cudaSuccess) e = cudaMemset(g_noalloc_ptr[d], 0, EX_NOALLOC_SCRATCH_BYTES);
    if (e != cudaSuccess && rc == EX_OK) rc = cuda_status(e);
  }
  e = cudaSetDevice(cur);
  if (e != cudaSuccess && rc == EX_OK) rc = cuda_status(e);
  return rc;
}

// 4-D tensor map over a paged K or V cache: (head dim, KV head, offset in page, page), 16-token x 64-dim boxes.
bool encode_kv_map(CUtensorMap* map, const void* base, int D, int KV, int BS, int64_t num_blocks, int64_t s_head,
                   int64_t s_page, int64_t s_block) {
  ex::PFN_encodeTiled enc = ex::get_encode_fn();
  if (!enc || reinterpret_cast<uintptr_t>(base) % 16 != 0) return false;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)KV, (cuuint64_t)BS, (cuuint64_t)num_blocks};
  cuuint64_t strides[3] = {(cuuint64_t)s_head * 2, (cuuint64_t)s_page * 2, (cuuint64_t)s_block * 2};
  cuuint32_t box[4] = {64, 1, 16, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_merge(const float* ws_m, const float* ws_l, const float* ws_acc, void* out, int64_t so_t, int64_t so_h,
                 int n, int H, int NS, int D, int out_dtype, const int32_t* seq_lens, int split, const int32_t* qsl,
                 cudaStream_t st) {
  const int mthreads = std::min(D, 256);
  const dim3 mg(n * H), mb(mthreads);
  cudaError_t e;
  if (out_dtype == EX_DTYPE_BF16)
    e = ex_launch_pdl(ex::k_paged_merge<EX_DTYPE_BF16>, mg, mb, 0, st, ws_m, ws_l, ws_acc, out, so_t, so_h, H, NS, D,
                      seq_lens, split, qsl);
  else if (out_dtype == EX_DTYPE_F16)
    e = ex_launch_pdl(ex::k_paged_merge<EX_DTYPE_F16>, mg, mb, 0, st, ws_m, ws_l, ws_acc, out, so_t, so_h, H, NS, D,
                      seq_lens, split, qsl);
  else
    e = ex_launch_pdl(ex::k_paged_merge<EX_DTYPE_F32>, mg, mb, 0, st, ws_m, ws_l, ws_acc, out, so_t, so_h, H, NS, D,
                      seq_lens, split, qsl);
  if (e != cudaSuccess) return cuda_status(e);
  return cuda_status(cudaGetLastError());
}

size_t linear_ws(int64_t M, int64_t N, int64_t K, int split_k, int algo) {
  if (M <= 0 || N <= 0) return 0;
  algo &= ~EX_LINEAR_STATIC_WEIGHTS;
  size_t a = simt_plan(M, N, K, split_k).ws_bytes;
  if (algo == EX_ALGO_SIMT) return a;
  const size_t b = ex::tc_plan(M, N, K, split_k, num_sms(), ex::tc_cluster_cap()).ws_bytes;
  if (algo == EX_ALGO_TC_I8) return b;
  return std::max(a, b);  // automatic choice: enough for either algorithm
}

// 4-D tensor map over a paged K or V cache of any element type for k_paged_rows: boxes of `box_rows` tokens of one
// page and head, `pitch` bytes of the head dimension wide.
bool encode_rows_map(CUtensorMap* map, const void* base, int esz, int D, int KV, int BS, int64_t num_blocks,
                     int64_t s_head, int64_t s_page, int64_t s_block, int pitch, int box_rows) {
  ex::PFN_encodeTiled enc = ex::get_encode_fn();
  if (!enc) return false;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)KV, (cuuint64_t)BS, (cuuint64_t)num_blocks};
  cuuint64_t strides[3] = {(cuuint64_t)s_head * esz, (cuuint64_t)s_page * esz, (cuuint64_t)s_block * esz};
  cuuint32_t box[4] = {(cuuint32_t)(pitch / esz), 1, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, esz == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(base),
             dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             pitch == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The stride of a dimension of one element says nothing (callers pass whatever their array type reports): D instead.
void one_element(int64_t size, int D, int64_t& stride) {
  if (size == 1) stride = D;
}
bool misaligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
bool half_dtype(int d) { return d == EX_DTYPE_BF16 || d == EX_DTYPE_F16; }
bool head_size_ok(int D) { return D == 64 || D == 128 || D == 256; }

// One launch of a kernel that takes dynamic shared memory, the attribute set once per device. regs > 0: its warps share out
// the registers of the launch and count on this many a thread (else cudaErrorNotSupported).
struct KernelReady {
  signed char dev[128] = {};  // 1: ready, -1: other registers than planned
};
template <typename K, typename... Args>
cudaError_t launch_smem(K kernel, KernelReady& ready, int regs, dim3 grid, int threads, int smem, cudaStream_t st,
                        const Args&... args) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 128) return cudaErrorNotSupported;
  if (ready.dev[dev] == 0) {
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    cudaFuncAttributes fa;
    if ((e = cudaFuncGetAttributes(&fa, kernel)) != cudaSuccess) return e;
    ready.dev[dev] = regs > 0 && fa.numRegs != regs ? -1 : 1;
  }
  if (ready.dev[dev] < 0) return cudaErrorNotSupported;
  return ex_launch_pdl(kernel, grid, dim3(threads), smem, st, args...);
}
int rows_status(cudaError_t e) { return e == cudaErrorNotSupported ? EX_ERR_UNSUPPORTED : cuda_status(e); }

template <int D, int CODE, bool F16, int NT>
cudaError_t launch_few_t(const CUtensorMap& mk, const CUtensorMap& mv, const ex::PrArgs& a, int64_t items,
                         cudaStream_t st) {
  using C = ex::PfCfg<D, CODE, NT>;
  static KernelReady ready;
  const int grid = (int)std::min<int64_t>(items, num_sms());
  return launch_smem(ex::k_paged_few<D, CODE, F16, NT>, ready, 0, dim3(grid), 32 * C::NW, C::SMEM, st, mk, mv, a);
}

// Requests of at most 16 rows a KV head go to k_paged_few, the others to k_tree_tc: by their own number of rows, so that
// a request's bits do not depend on the longest one of the batch.
template <int D, int CODE, bool F16>
cudaError_t launch_rows_nt(int rows, const CUtensorMap& mk, const CUtensorMap& mv, ex::PrArgs a,
                           int64_t per_tile, cudaStream_t st) {
  a.rows_lo = 0;
  a.rows_hi = ex::PR_FEW;
  if (rows <= 8) return launch_few_t<D, CODE, F16, 1>(mk, mv, a, per_tile, st);
  if (rows <= ex::PR_FEW) return launch_few_t<D, CODE, F16, 2>(mk, mv, a, per_tile, st);
  const cudaError_t e = launch_few_t<D, CODE, F16, 2>(mk, mv, a, per_tile, st);  // (how many there are is known on the device)
  if (e != cudaSuccess) return e;
  a.rows_lo = ex::PR_FEW;
  a.rows_hi = INT32_MAX;
  using C = ex::PtcCfg<D, CODE>;
  static KernelReady ready;
  const int grid = (int)std::min<int64_t>(per_tile * cdiv(rows, 128), num_sms());
  return launch_smem(ex::k_tree_tc<D, CODE, F16>, ready, C::REGS, dim3(grid), C::THREADS, C::SMEM, st, mk, mv, a);
}

template <int D>
cudaError_t launch_rows_d(int code, int q_dtype, int rows, const CUtensorMap& mk, const CUtensorMap& mv,
                          const ex::PrArgs& a, int64_t per_tile, cudaStream_t st) {
  cudaError_t e;
  if (code == ex::CODE_INT8) e = launch_rows_nt<D, ex::CODE_INT8, true>(rows, mk, mv, a, per_tile, st);
  else if (code == ex::CODE_E4M3) e = launch_rows_nt<D, ex::CODE_E4M3, true>(rows, mk, mv, a, per_tile, st);
  else if (q_dtype == EX_DTYPE_F16) e = launch_rows_nt<D, ex::CODE_NONE, true>(rows, mk, mv, a, per_tile, st);
  else e = launch_rows_nt<D, ex::CODE_NONE, false>(rows, mk, mv, a, per_tile, st);
  if (e != cudaSuccess || a.NS == 1) return e;
  const dim3 grid((unsigned)cdiv(a.tokens * a.H * (D / 64), 4)), block(128);
  if (q_dtype == EX_DTYPE_F16) return ex_launch_pdl(ex::k_paged_rows_merge<D, true>, grid, block, 0, st, a);
  return ex_launch_pdl(ex::k_paged_rows_merge<D, false>, grid, block, 0, st, a);
}

// ex_paged_decode_q8 and ex_tree_attention: checks, tensor maps, launches.
int paged_rows(const void* q, int64_t sq_t, int64_t sq_h, int q_dtype, const void* k_cache, const void* v_cache, int code,
               int64_t s_block, int64_t s_page, int64_t s_head, const float* k_scale, const float* v_scale,
               int64_t ss_block, int64_t ss_head, int64_t num_blocks, const int32_t* block_table, int64_t sbt, int width,
               const int32_t* seq_lens, const int32_t* qsl, const int64_t* mask, int n, int64_t tokens, int max_tokens,
               int H, int KV, int D, int BS, float scale, int64_t max_len, void* out, int64_t so_t, int64_t so_h,
               void* workspace, size_t workspace_bytes, cudaStream_t st) {
  if (n < 0 || tokens < 0 || tokens > INT32_MAX || H <= 0 || KV <= 0 || H % KV != 0 || BS <= 0 || width < 0 || max_len < 0)
    return EX_ERR_ARG;
  if (code < ex::CODE_NONE || code > ex::CODE_E4M3 || max_tokens < 1) return EX_ERR_ARG;
  // (0 times the -infinity of a key that is not seen would be NaN)
  if (!(fabsf(scale) > 0.0f && fabsf(scale * ex::PR_LOG2E) < INFINITY)) return EX_ERR_ARG;
  if (!half_dtype(q_dtype)) return EX_ERR_DTYPE;
  const int G = H / KV;
  if (G > 16 || !head_size_ok(D) || BS % 8 != 0 || max_tokens > ex::PR_MAX_TOKENS) return EX_ERR_UNSUPPORTED;
  if (n == 0 || tokens == 0) return EX_OK;
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out || num_blocks <= 0) return EX_ERR_ARG;
  if (code != ex::CODE_NONE && (!k_scale || !v_scale)) return EX_ERR_ARG;
  for (int64_t* s : {&sq_t, &so_t}) one_element(tokens, D, *s);
  for (int64_t* s : {&sq_h, &so_h}) one_element(H, D, *s);
  for (int64_t* s : {&s_head, &ss_head}) one_element(KV, D, *s);
  for (int64_t* s : {&s_block, &ss_block}) one_element(num_blocks, D, *s);
  const int esz = code == ex::CODE_NONE ? 2 : 1, vec = 16 / esz;
  if (misaligned(q, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(out, 4) || sq_t % 8 != 0 ||
      sq_h % 8 != 0 || s_block % vec != 0 || s_page % vec != 0 || s_head % vec != 0 || so_t % 2 != 0 || so_h % 2 != 0)
    return EX_ERR_ALIGN;
  if (code != ex::CODE_NONE && (misaligned(k_scale, 16) || misaligned(v_scale, 16) || ss_block % 4 != 0 || ss_head % 4 != 0))
    return EX_ERR_ALIGN;
  max_len = std::min<int64_t>(max_len, std::min<int64_t>((int64_t)width * BS, INT32_MAX - 4096));
  const int NS = ex::pr_max_segments(max_len);
  const int64_t rows = tokens * H * NS;
  const size_t need = ex_paged_rows_workspace_bytes(tokens, H, D, max_len);
  if (need > 0 && (!workspace || workspace_bytes < need)) return EX_ERR_WORKSPACE;
  if (need > 0 && misaligned(workspace, 256)) return EX_ERR_ALIGN;
  const int per_tile_rows = max_tokens * G;
  const int64_t per_tile = (int64_t)n * NS * KV;
  if (per_tile * cdiv(per_tile_rows, 8) > INT32_MAX) return EX_ERR_UNSUPPORTED;  // items are numbered in 32 bits
  if (!ex::device_is_sm100()) return EX_ERR_UNSUPPORTED;
  ex::PrArgs a = {};
  a.q = q; a.sq_t = sq_t; a.sq_h = sq_h; a.q_is_f16 = q_dtype == EX_DTYPE_F16;
  a.bt = block_table; a.sbt = sbt; a.seq_lens = seq_lens; a.qsl = qsl;
  a.mask = reinterpret_cast<const uint64_t*>(mask);
  a.n = n; a.H = H; a.G = G; a.g_inv = (65536u + G - 1) / G; a.KV = KV; a.BS = BS; a.group_log2 = BS % 16 == 0 ? 4 : 3; a.max_tokens = max_tokens;
  a.max_keys = (int)max_len; a.blocks = num_blocks; a.tokens = tokens; a.scale_log2 = scale * ex::PR_LOG2E;
  a.k_scale = k_scale; a.v_scale = v_scale; a.ss_block = ss_block; a.ss_head = ss_head; a.NS = NS;
  a.v = v_cache; a.sv_block = s_block; a.sv_page = s_page; a.sv_head = s_head;
  if (need > 0) {
    char* w = reinterpret_cast<char*>(workspace);
    a.ws_m = reinterpret_cast<float*>(w);
    a.ws_l = reinterpret_cast<float*>(w + align_up((size_t)rows * 4, 256));
    a.ws_acc = reinterpret_cast<float*>(w + 2 * align_up((size_t)rows * 4, 256));
  }
  a.out = out; a.so_t = so_t; a.so_h = so_h;
  const int pitch = std::min(128, D * esz), box = 1 << a.group_log2;
  CUtensorMap mk, mv;
  if (!encode_rows_map(&mk, k_cache, esz, D, KV, BS, num_blocks, s_head, s_page, s_block, pitch, box) ||
      !encode_rows_map(&mv, v_cache, esz, D, KV, BS, num_blocks, s_head, s_page, s_block, pitch, box))
    return EX_ERR_UNSUPPORTED;
  cudaError_t e;
  if (D == 64) e = launch_rows_d<64>(code, q_dtype, per_tile_rows, mk, mv, a, per_tile, st);
  else if (D == 128) e = launch_rows_d<128>(code, q_dtype, per_tile_rows, mk, mv, a, per_tile, st);
  else e = launch_rows_d<256>(code, q_dtype, per_tile_rows, mk, mv, a, per_tile, st);
  return rows_status(e);
}

// 3-D tensor map over packed rows (D, heads, rows): boxes of 128 rows of one head, 64 dims wide.
bool encode_packed_map(CUtensorMap* map, const void* base, int D, int heads, int64_t rows, int64_t s_h, int64_t s_t) {
  ex::PFN_encodeTiled enc = ex::get_encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)s_h * 2, (cuuint64_t)s_t * 2};
  cuuint32_t box[3] = {64, 1, 128};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool F16>
int launch_prompt(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, ex::PaArgs a, cudaStream_t st) {
  using C = ex::PaCfg<D>;
  static KernelReady ready;
  a.tiles = (int)(cdiv(a.tokens, C::ROWS) + a.n);  // at least as many as there are
  if ((int64_t)a.tiles * a.H > INT32_MAX) return EX_ERR_UNSUPPORTED;
  return rows_status(launch_smem(ex::k_prompt_attn<D, F16>, ready, ex::PA_REGS_LAUNCH, dim3((unsigned)(a.tiles * a.H)),
                                 ex::PA_THREADS, C::SMEM, st, mq, mk, mv, a));
}

template <int D, int CODE, int PASSES, typename T>
cudaError_t launch_cache_write_t(const void* key, const void* value, int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h,
                                 const ex::CacheView& c, const int64_t* slots, int64_t tokens, int KV, void* ko, void* vo,
                                 int64_t sko_t, int64_t sko_h, int64_t svo_t, int64_t svo_h, cudaStream_t st) {
  const int64_t per_token = cdiv(2 * KV, (32 / (D / 8)) * PASSES), items = tokens * per_token;  // a warp each
  const dim3 grid((unsigned)cdiv(items, ex::CQ_THREADS / 32)), block(ex::CQ_THREADS);
  return ex_launch_pdl(ex::k_cache_write<D, CODE, T, PASSES>, grid, block, 0, st, (const T*)key, (const T*)value, sk_t, sk_h,
                       sv_t, sv_h, c, slots, (uint32_t)items, (uint32_t)per_token, KV, (T*)ko, (T*)vo, sko_t, sko_h, svo_t, svo_h);
}
template <int D, int CODE, typename T>
cudaError_t launch_cache_write(const void* key, const void* value, int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h,
                               const ex::CacheView& c, const int64_t* slots, int64_t tokens, int KV, void* ko, void* vo,
                               int64_t sko_t, int64_t sko_h, int64_t svo_t, int64_t svo_h, cudaStream_t st) {
  // one pass a warp while that leaves no warp waiting (64 of an SM run at once)
  const bool few = tokens * cdiv(2 * KV, 32 / (D / 8)) <= 64 * (int64_t)num_sms();
  return (few ? launch_cache_write_t<D, CODE, 1, T> : launch_cache_write_t<D, CODE, 4, T>)(
      key, value, sk_t, sk_h, sv_t, sv_h, c, slots, tokens, KV, ko, vo, sko_t, sko_h, svo_t, svo_h, st);
}

template <int D, int CODE>
cudaError_t launch_cache_read(const ex::CacheView& c, const int32_t* bt, int64_t sbt, int width, const int32_t* cu, int n,
                              int64_t rows, int KV, int f16, void* ko, void* vo, int64_t sko_t, int64_t sko_h,
                              int64_t svo_t, int64_t svo_h, cudaStream_t st) {
  const dim3 grid((unsigned)cdiv(rows, ex::CQ_THREADS / 32)), block(ex::CQ_THREADS);
  if (f16)
    return ex_launch_pdl(ex::k_cache_read<D, CODE, __half>, grid, block, 0, st, c, bt, sbt, width, cu, n, rows, KV,
                         (__half*)ko, (__half*)vo, sko_t, sko_h, svo_t, svo_h);
  return ex_launch_pdl(ex::k_cache_read<D, CODE, __nv_bfloat16>, grid, block, 0, st, c, bt, sbt, width, cu, n, rows, KV,
                       (__nv_bfloat16*)ko, (__nv_bfloat16*)vo, sko_t, sko_h, svo_t, svo_h);
}

// Shared checks of the two cache entry points.
int check_cache(int dtype, int code, const void* k_cache, const void* v_cache, int64_t& s_block, int64_t& s_page,
                int64_t& s_head, const float* k_scale, const float* v_scale, int64_t num_blocks, int BS, int KV, int D) {
  if (KV <= 0 || BS <= 0 || num_blocks <= 0 || code < ex::CODE_INT8 || code > ex::CODE_E4M3) return EX_ERR_ARG;
  if (!half_dtype(dtype)) return EX_ERR_DTYPE;
  if (!head_size_ok(D)) return EX_ERR_UNSUPPORTED;
  if (!k_cache || !v_cache || !k_scale || !v_scale) return EX_ERR_ARG;
  one_element(KV, D, s_head);
  one_element(BS, D, s_page);
  one_element(num_blocks, D, s_block);
  if (misaligned(k_cache, 16) || misaligned(v_cache, 16) || s_block % 16 != 0 || s_page % 16 != 0 || s_head % 16 != 0 ||
      misaligned(k_scale, 4) || misaligned(v_scale, 4))
    return EX_ERR_ALIGN;
  return EX_OK;
}

ex::CacheView cache_view(const void* k, const void* v, int64_t s_block, int64_t s_page, int64_t s_head, const float* ks,
                         const float* vs, int64_t ss_block, int64_t ss_head, int64_t blocks, int BS) {
  ex::CacheView c;
  c.key = (uint8_t*)const_cast<void*>(k); c.value = (uint8_t*)const_cast<void*>(v);
  c.s_block = s_block; c.s_page = s_page; c.s_head = s_head;
  c.key_scale = const_cast<float*>(ks); c.value_scale = const_cast<float*>(vs);
  c.ss_block = ss_block; c.ss_head = ss_head; c.blocks = blocks; c.page = BS;
  return c;
}

}  // namespace

extern "C" {

const char* ex_version(void) { return "vllm-exact-b200 0.1.0 (sm_100a)"; }

const char* ex_status_string(int s) {
  switch (s) {
    case EX_OK: return "ok";
    case EX_ERR_ARG: return "invalid argument";
    case EX_ERR_ALIGN: return "misaligned pointer or leading dimension";
    case EX_ERR_WORKSPACE: return "workspace missing or too small";
    case EX_ERR_DTYPE: return "unsupported dtype";
    case EX_ERR_UNSUPPORTED: return "unsupported shape or algorithm";
    case EX_ERR_CUDA: return "CUDA error";
    case EX_ERR_DEVICE: return "device-side bounded wait timed out";
    default: return "unknown status";
  }
}

const char* ex_last_error_string(void) { return g_last_error.c_str(); }

int ex_device_error(int* code) {
  if (!code) return EX_ERR_ARG;
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return cuda_status(e);
  int v = 0;
  e = cudaMemcpyFromSymbol(&v, g_ex_dev_error, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e);
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_ex_dev_error, &zero, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e);
  *code = v;
  if (v != 0) return noalloc_clear_all();  // a stopped call may have left the static split-K scratch dirty
  return EX_OK;
}

int ex_digitize(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t K, int F, int8_t* h, int8_t* l,
                int64_t ldd, int32_t* cs, int32_t* sh, void* stream) {
  if (rows < 0 || K < 0 || rows > INT32_MAX || K > INT32_MAX) return EX_ERR_ARG;
  if (F != 14 && F != 15) return EX_ERR_ARG;
  if (!dtype_ok(x_dtype)) return EX_ERR_DTYPE;
  if (rows == 0) return EX_OK;
  if (!cs || !sh) return EX_ERR_ARG;
  if (K > 0 && (!x || !h || !l || ldx < K || ldd < K)) return EX_ERR_ARG;
  return cuda_status(
      ex::launch_digitize<ex::DIG_LOCAL>(x, x_dtype, ldx, rows, K, F, h, l, ldd, cs, sh, nullptr, (cudaStream_t)stream));
}

int ex_row_absmax(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t K, float* amax, void* stream) {
  if (rows < 0 || K < 0 || rows > INT32_MAX || K > INT32_MAX) return EX_ERR_ARG;
  if (!dtype_ok(x_dtype)) return EX_ERR_DTYPE;
  if (rows == 0) return EX_OK;
  if (!amax || (K > 0 && (!x || ldx < K))) return EX_ERR_ARG;
  return cuda_status(ex::launch_digitize<ex::DIG_ABSMAX>(x, x_dtype, ldx, rows, K, 14, nullptr, nullptr, K, nullptr,
                                                         nullptr, amax, (cudaStream_t)stream));
}

int ex_digitize_given_absmax(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t K, int F,
                             const float* amax, int8_t* h, int8_t* l, int64_t ldd, int32_t* cs, int32_t* sh,
                             void* stream) {
  if (rows < 0 || K < 0 || rows > INT32_MAX || K > INT32_MAX) return EX_ERR_ARG;
  if (F != 14 && F != 15) return EX_ERR_ARG;
  if (!dtype_ok(x_dtype)) return EX_ERR_DTYPE;
  if (rows == 0) return EX_OK;
  if (!cs || !sh || !amax) return EX_ERR_ARG;
  if (K > 0 && (!x || !h || !l || ldx < K || ldd < K)) return EX_ERR_ARG;
  return cuda_status(ex::launch_digitize<ex::DIG_GIVEN>(x, x_dtype, ldx, rows, K, F, h, l, ldd, cs, sh,
                                                        const_cast<float*>(amax), (cudaStream_t)stream));
}

size_t ex_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int split_k, int algo) {
  return linear_ws(M, N, K, split_k, algo);
}

int ex_linear(const int8_t* xh, const int8_t* xl, int64_t ldx, const int32_t* cx, const int32_t* sx,
              const int8_t* wh, const int8_t* wl, int64_t ldw, const int32_t* cw, const int32_t* sw, int64_t M,
              int64_t N, int64_t K, int F, int trunc, void* out, int out_dtype, int64_t ldo, void* workspace,
              size_t workspace_bytes, int split_k, int algo, void* stream) {
  return linear_impl<false>(xh, xl, ldx, cx, sx, wh, wl, ldw, cw, sw, M, N, K, F, trunc, out, out_dtype, ldo,
                            workspace, workspace_bytes, split_k, algo, (cudaStream_t)stream);
}

int ex_linear_noalloc(const int8_t* xh, const int8_t* xl, int64_t ldx, const int32_t* cx, const int32_t* sx,
                      const int8_t* wh, const int8_t* wl, int64_t ldw, const int32_t* cw, const int32_t* sw,
                      int64_t M, int64_t N, int64_t K, int F, int trunc, void* out, int out_dtype, int64_t ldo,
                      int split_k, int algo, void* stream) {
  int rc = check_linear_args(xh, xl, ldx, cx, wh, wl, ldw, cw, M, N, K, F, out, ldo);
  if (rc != EX_OK || M == 0 || N == 0) return rc;
  if (split_k < 0) return EX_ERR_ARG;
  const int chosen = pick_algo(algo & ~EX_LINEAR_STATIC_WEIGHTS, xh, xl, ldx, wh, wl, ldw, M, N, K);
  size_t need = 0;
  if (chosen == EX_ALGO_SIMT)
    need = simt_plan(M, N, K, split_k).ws_bytes;
  else if (chosen == EX_ALGO_TC_I8 && ex::tc_supported(xh, xl, ldx, wh, wl, ldw, M, N, K))
    need = ex::tc_plan(M, N, K, split_k, num_sms(), ex::tc_cluster_cap()).ws_bytes;
  if (need > EX_NOALLOC_SCRATCH_BYTES) {
    g_last_error = "ex_linear_noalloc: this shape's split-K plan needs " + std::to_string(need) +
                   " bytes of scratch, more than the static EX_NOALLOC_SCRATCH_BYTES (" +
                   std::to_string((size_t)EX_NOALLOC_SCRATCH_BYTES) + ")";
    return EX_ERR_WORKSPACE;
  }
  void* scratch = nullptr;
  rc = noalloc_scratch((cudaStream_t)stream, &scratch);
  if (rc != EX_OK) return rc;
  return linear_impl<false>(xh, xl, ldx, cx, sx, wh, wl, ldw, cw, sw, M, N, K, F, trunc, out, out_dtype, ldo, scratch,
                            EX_NOALLOC_SCRATCH_BYTES, split_k, algo, (cudaStream_t)stream);
}

int ex_linear_noalloc_reset(void* stream) {
  void* scratch = nullptr;
  const int rc = noalloc_scratch((cudaStream_t)stream, &scratch);
  if (rc != EX_OK) return rc;
  return cuda_status(cudaMemsetAsync(scratch, 0, EX_NOALLOC_SCRATCH_BYTES, (cudaStream_t)stream));
}

int ex_linear_noalloc_fill_scratch(int byte_value, void* stream) {
  if (byte_value < 0 || byte_value > 255) return EX_ERR_ARG;
  void* scratch = nullptr;
  const int rc = noalloc_scratch((cudaStream_t)stream, &scratch);
  if (rc != EX_OK) return rc;
  return cuda_status(cudaMemsetAsync(scratch, byte_value, EX_NOALLOC_SCRATCH_BYTES, (cudaStream_t)stream));
}

int ex_linear_partial_i64(const int8_t* xh, const int8_t* xl, int64_t ldx, const int32_t* cx, const int8_t* wh,
                          const int8_t* wl, int64_t ldw, const int32_t* cw, int64_t M, int64_t N, int64_t K, int F,
                          int trunc, int64_t* tot, int64_t ldt, void* workspace, size_t workspace_bytes, int split_k,
                          int algo, void* stream) {
  return linear_impl<true>(xh, xl, ldx, cx, nullptr, wh, wl, ldw, cw, nullptr, M, N, K, F, trunc, tot,
                           EX_DTYPE_F32, ldt, workspace, workspace_bytes, split_k, algo, (cudaStream_t)stream);
}

int ex_epilogue_i64(const int64_t* tot, int64_t ldt, const int32_t* sx, const int32_t* sw, int64_t M, int64_t N,
                    void* out, int out_dtype, int64_t ldo, void* stream) {
  if (M < 0 || N < 0 || M > INT32_MAX || N > INT32_MAX) return EX_ERR_ARG;
  if (!dtype_ok(out_dtype)) return EX_ERR_DTYPE;
  if (M == 0 || N == 0) return EX_OK;
  if (!tot || !sx || !sw || !out || ldt < N || ldo < N) return EX_ERR_ARG;
  const int64_t total = M * N;
  const int threads = 256;
  const int blocks = (int)std::min<int64_t>(cdiv(total, threads), 16 * (int64_t)num_sms());
  cudaStream_t st = (cudaStream_t)stream;
  const long long* t = reinterpret_cast<const long long*>(tot);
  if (out_dtype == EX_DTYPE_F32)
    ex::k_epilogue_i64<EX_DTYPE_F32><<<blocks, threads, 0, st>>>(t, ldt, sx, sw, (int)M, (int)N, out, ldo);
  else if (out_dtype == EX_DTYPE_BF16)
    ex::k_epilogue_i64<EX_DTYPE_BF16><<<blocks, threads, 0, st>>>(t, ldt, sx, sw, (int)M, (int)N, out, ldo);
  else
    ex::k_epilogue_i64<EX_DTYPE_F16><<<blocks, threads, 0, st>>>(t, ldt, sx, sw, (int)M, (int)N, out, ldo);
  return cuda_status(cudaGetLastError());
}

int ex_ipc_get_handle(const void* dev_ptr, unsigned char* handle, uint64_t* offset) {
  if (!dev_ptr || !handle || !offset) return EX_ERR_ARG;
  typedef CUresult (*PFN_range)(CUdeviceptr*, size_t*, CUdeviceptr);
  static PFN_range range_fn = nullptr;
  if (!range_fn) {
    void* fp = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuMemGetAddressRange", &fp, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return EX_ERR_UNSUPPORTED;
    range_fn = reinterpret_cast<PFN_range>(fp);
  }
  CUdeviceptr base = 0;
  size_t size = 0;
  if (range_fn(&base, &size, reinterpret_cast<CUdeviceptr>(dev_ptr)) != CUDA_SUCCESS) return EX_ERR_ARG;
  cudaIpcMemHandle_t h;
  cudaError_t e = cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base));
  if (e != cudaSuccess) return cuda_status(e);
  static_assert(sizeof(h) == EX_IPC_HANDLE_BYTES, "IPC handle size");
  std::memcpy(handle, &h, sizeof(h));
  *offset = (uint64_t)(reinterpret_cast<CUdeviceptr>(dev_ptr) - base);
  return EX_OK;
}

int ex_ipc_open_handle(const unsigned char* handle, void** base) {
  if (!handle || !base) return EX_ERR_ARG;
  cudaIpcMemHandle_t h;
  std::memcpy(&h, handle, sizeof(h));
  return cuda_status(cudaIpcOpenMemHandle(base, h, cudaIpcMemLazyEnablePeerAccess));
}

int ex_ipc_close_handle(void* base) {
  if (!base) return EX_ERR_ARG;
  return cuda_status(cudaIpcCloseMemHandle(base));
}

int ex_tp_digitize(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t K, int F, const void* xch,
                   int64_t max_rows, int32_t* ctl, int rank, int world, int8_t* h, int8_t* l, int64_t ldd, int32_t* cs,
                   int32_t* sh, void* stream) {
  if (rows < 0 || K < 0 || rows > INT32_MAX || K > INT32_MAX || max_rows > INT32_MAX) return EX_ERR_ARG;
  if (F != 14 && F != 15) return EX_ERR_ARG;
  if (!dtype_ok(x_dtype)) return EX_ERR_DTYPE;
  if (world < 1 || world > ex::TPF_MAX_WORLD || rank < 0 || rank >= world) return EX_ERR_ARG;
  if (!xch || !ctl || rows > max_rows) return EX_ERR_ARG;
  if (rows == 0) return EX_OK;  // every rank makes the same call, so every rank skips it
  if (!cs || !sh || (K > 0 && (!x || !h || !l || ldx < K || ldd < K))) return EX_ERR_ARG;
  // all blocks resident together (256 threads, no dynamic shared memory): every wait is on other ranks only
  const int blocks = (int)std::min<int64_t>(rows, 4 * (int64_t)num_sms());
  cudaStream_t st = (cudaStream_t)stream;
  unsigned long long* const* xp = reinterpret_cast<unsigned long long* const*>(xch);
  cudaError_t e = cudaSuccess;
#define EX_TPD(T, FF)                                                                                              \
  e = ex_launch_pdl(ex::k_tp_digitize<T, FF>, dim3(blocks), dim3(ex::DIG_THREADS), 0, st,                          \
                    reinterpret_cast<const T*>(x), ldx, (int)rows, (int)K, xp, ctl, rank, world, (int)max_rows, h, l, \
                    ldd, cs, sh)
  if (x_dtype == EX_DTYPE_F32) {
    if (F == 15) EX_TPD(float, 15); else EX_TPD(float, 14);
  } else if (x_dtype == EX_DTYPE_BF16) {
    if (F == 15) EX_TPD(__nv_bfloat16, 15); else EX_TPD(__nv_bfloat16, 14);
  } else {
    if (F == 15) EX_TPD(__half, 15); else EX_TPD(__half, 14);
  }
#undef EX_TPD
  return cuda_status(e);
}

int ex_allreduce_epilogue_i64(const void* parts, int64_t ldt, const void* xch, const void* flags, int32_t* ctl,
                              int rank, int world, const int32_t* sx, const int32_t* sw, int64_t M, int64_t N,
                              void* out, int out_dtype, int64_t ldo, void* stream) {
  if (M < 0 || N < 0 || M > INT32_MAX || N > INT32_MAX) return EX_ERR_ARG;
  if (world < 1 || world > ex::TPF_MAX_WORLD || rank < 0 || rank >= world) return EX_ERR_ARG;
  if (!dtype_ok(out_dtype)) return EX_ERR_DTYPE;
  if (!parts || !xch || !flags || !ctl || !sx || !sw || !out || ldt < N || ldo < N) return EX_ERR_ARG;
  if (N % 2 != 0 || ldt % 2 != 0 || ldo % 2 != 0) return EX_ERR_ALIGN;  // column pairs: 16-byte partial loads
  // every rank takes part in every call, also for an empty output (one block then only exchanges the flags). The
  // block count depends on (M, N, world) only, so it is the same on every rank: block b pairs with block b of the
  // others; at most TPF_MAX_BLOCKS small blocks, all resident together.
  const int64_t pairs = M * cdiv(N, 2 * (int64_t)world);
  const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(pairs, ex::TPF_THREADS), ex::TPF_MAX_BLOCKS));
  cudaStream_t st = (cudaStream_t)stream;
  const long long* const* pp = reinterpret_cast<const long long* const*>(parts);
  unsigned long long* const* xp = reinterpret_cast<unsigned long long* const*>(xch);
  int* const* fp = reinterpret_cast<int* const*>(flags);
  cudaError_t e;
#define EX_TPF_LAUNCH(OD)                                                                                        \
  e = ex_launch_pdl(ex::k_tp_allreduce_epilogue<OD>, dim3(blocks), dim3(ex::TPF_THREADS), 0, st, pp, ldt, xp, fp, \
                    ctl, rank, world, sx, sw, (int)M, (int)N, out, ldo)
  if (out_dtype == EX_DTYPE_F32)
    EX_TPF_LAUNCH(EX_DTYPE_F32);
  else if (out_dtype == EX_DTYPE_BF16)
    EX_TPF_LAUNCH(EX_DTYPE_BF16);
  else
    EX_TPF_LAUNCH(EX_DTYPE_F16);
#undef EX_TPF_LAUNCH
  return cuda_status(e);
}

size_t ex_paged_decode_workspace_bytes(int n, int H, int D, int max_len, int split) {
  if (n <= 0 || H <= 0 || D <= 0 || split <= 0) return 0;
  const int64_t NS = std::max<int64_t>(1, cdiv(max_len, split));
  const int64_t rows = (int64_t)n * H * NS;
  return align_up((size_t)rows * 4, 256) * 2 + (size_t)rows * D * 4;
}

int ex_paged_decode(const void* q, int64_t sq_t, int64_t sq_h, const void* k_cache, const void* v_cache,
                    int64_t s_block, int64_t s_page, int64_t s_head, int64_t num_blocks, const int32_t* block_table,
                    int64_t sbt,
                    const int32_t* seq_lens, int n, int H, int KV, int D, int BS, float scale, int max_len, int split,
                    void* out, int64_t so_t, int64_t so_h, int out_dtype, void* workspace, size_t workspace_bytes,
                    void* stream) {
  return ex_paged_decode_leading(q, sq_t, sq_h, k_cache, v_cache, s_block, s_page, s_head, num_blocks, block_table,
                                 sbt, seq_lens, nullptr, n, H, KV, D, BS, scale, max_len, split, out, so_t, so_h,
                                 out_dtype, workspace, workspace_bytes, stream);
}

int ex_paged_decode_leading(const void* q, int64_t sq_t, int64_t sq_h, const void* k_cache, const void* v_cache,
                            int64_t s_block, int64_t s_page, int64_t s_head, int64_t num_blocks,
                            const int32_t* block_table, int64_t sbt, const int32_t* seq_lens,
                            const int32_t* query_start_loc, int n, int H, int KV, int D, int BS, float scale,
                            int max_len, int split, void* out, int64_t so_t, int64_t so_h, int out_dtype,
                            void* workspace, size_t workspace_bytes, void* stream) {
  if (n < 0 || H <= 0 || KV <= 0 || H % KV != 0 || BS <= 0 || split <= 0 || max_len < 0) return EX_ERR_ARG;
  const int G = H / KV;
  if (G > 16) return EX_ERR_UNSUPPORTED;
  if (D != 64 && D != 128 && D != 256) return EX_ERR_UNSUPPORTED;
  if (!dtype_ok(out_dtype)) return EX_ERR_DTYPE;
  if (n == 0) return EX_OK;
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out) return EX_ERR_ARG;
  // 16-byte cp.async gathers and 4-byte query loads
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) % 16 != 0 ||
      s_block % 8 != 0 || s_page % 8 != 0 || s_head % 8 != 0)
    return EX_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(q) % 4 != 0 || sq_t % 2 != 0 || sq_h % 2 != 0) return EX_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(query_start_loc) % 4 != 0) return EX_ERR_ALIGN;
  const size_t need = ex_paged_decode_workspace_bytes(n, H, D, max_len, split);
  if (!workspace || workspace_bytes < need) return EX_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return EX_ERR_ALIGN;
  const int NS = (int)std::max<int64_t>(1, cdiv(max_len, split));
  if (KV > 65535 || NS > 65535) return EX_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)n * H * NS;
  float* ws_m = reinterpret_cast<float*>(workspace);
  float* ws_l = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + align_up((size_t)rows * 4, 256));
  float* ws_acc = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + 2 * align_up((size_t)rows * 4, 256));
  cudaStream_t st = (cudaStream_t)stream;
  const __nv_bfloat16* qp = reinterpret_cast<const __nv_bfloat16*>(q);
  const __nv_bfloat16* kp = reinterpret_cast<const __nv_bfloat16*>(k_cache);
  const __nv_bfloat16* vp = reinterpret_cast<const __nv_bfloat16*>(v_cache);
  dim3 grid(n, KV, NS);
  cudaError_t e = cudaSuccess;
  if (num_blocks <= 0) return EX_ERR_ARG;
  // TMA page-gather kernel for the common layouts; the cp.async kernel below handles everything else
  if ((D == 64 || D == 128) && G <= 8 && BS % 16 == 0 && split % ex::PT_BLK == 0 && ex::device_is_sm100()) {
    CUtensorMap mk, mv;
    if (encode_kv_map(&mk, k_cache, D, KV, BS, num_blocks, s_head, s_page, s_block) &&
        encode_kv_map(&mv, v_cache, D, KV, BS, num_blocks, s_head, s_page, s_block)) {
      const dim3 blk(ex::PT_THREADS);
#define EX_PT_LAUNCH(DD)                                                                                         \
  {                                                                                                              \
    const int smem = ex::PtCfg<DD>::SMEM;                                                                        \
    e = cudaFuncSetAttribute(ex::k_paged_tma<DD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);            \
    if (e == cudaSuccess)                                                                                        \
      e = ex_launch_pdl(ex::k_paged_tma<DD>, grid, blk, smem, st, mk, mv, qp, sq_t, sq_h, block_table, sbt,      \
                        seq_lens, query_start_loc, H, G, BS, scale, split, NS, ws_m, ws_l, ws_acc);              \
  }
      if (D == 64) EX_PT_LAUNCH(64)
      else EX_PT_LAUNCH(128)
#undef EX_PT_LAUNCH
      if (e != cudaSuccess) return cuda_status(e);
      return launch_merge(ws_m, ws_l, ws_acc, out, so_t, so_h, n, H, NS, D, out_dtype, seq_lens, split,
                        query_start_loc, st);
    }
  }
#define EX_PD_LAUNCH(DD)                                                                                         \
  {                                                                                                              \
    const int smem = ex::PdCfg<DD>::SMEM;                                                                        \
    e = cudaFuncSetAttribute(ex::k_paged_partial<DD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);        \
    if (e == cudaSuccess)                                                                                        \
      e = ex_launch_pdl(ex::k_paged_partial<DD>, grid, dim3(ex::PD_THREADS), smem, st, qp, sq_t, sq_h, kp, vp,   \
                        s_block, s_page, s_head, block_table, sbt, seq_lens, query_start_loc, H, G, BS, scale,   \
                        split, NS, ws_m, ws_l, ws_acc);                                                          \
  }
  if (D == 64) EX_PD_LAUNCH(64)
  else if (D == 128) EX_PD_LAUNCH(128)
  else EX_PD_LAUNCH(256)
#undef EX_PD_LAUNCH
  if (e != cudaSuccess) return cuda_status(e);
  if ((e = cudaGetLastError()) != cudaSuccess) return cuda_status(e);
  return launch_merge(ws_m, ws_l, ws_acc, out, so_t, so_h, n, H, NS, D, out_dtype, seq_lens, split,
                        query_start_loc, st);
}

size_t ex_paged_rows_workspace_bytes(int64_t tokens, int H, int D, int64_t max_len) {
  if (tokens <= 0 || H <= 0 || D <= 0 || max_len < 0) return 0;
  const int64_t NS = ex::pr_max_segments(std::min<int64_t>(max_len, INT32_MAX - 4096));
  if (NS == 1) return 0;
  const size_t rows = (size_t)tokens * H * NS;
  return align_up(rows * 4, 256) * 2 + rows * D * 4;
}

int ex_paged_decode_q8(const void* q, int64_t sq_t, int64_t sq_h, int q_dtype, const void* k_cache, const void* v_cache,
                       int code, int64_t s_block, int64_t s_page, int64_t s_head, const float* k_scale,
                       const float* v_scale, int64_t ss_block, int64_t ss_head, int64_t num_blocks,
                       const int32_t* block_table, int64_t sbt, int width, const int32_t* seq_lens, int n, int H, int KV,
                       int D, int BS, float scale, int64_t max_len, void* out, int64_t so_t, int64_t so_h,
                       void* workspace, size_t workspace_bytes, void* stream) {
  if (code == EX_CODE_NONE) return EX_ERR_ARG;
  return paged_rows(q, sq_t, sq_h, q_dtype, k_cache, v_cache, code, s_block, s_page, s_head, k_scale, v_scale, ss_block,
                    ss_head, num_blocks, block_table, sbt, width, seq_lens, nullptr, nullptr, n, n, 1, H, KV, D, BS,
                    scale, max_len, out, so_t, so_h, workspace, workspace_bytes, (cudaStream_t)stream);
}

int ex_tree_attention(const void* q, int64_t sq_t, int64_t sq_h, int q_dtype, const void* k_cache, const void* v_cache,
                      int code, int64_t s_block, int64_t s_page, int64_t s_head, const float* k_scale,
                      const float* v_scale, int64_t ss_block, int64_t ss_head, int64_t num_blocks,
                      const int32_t* block_table, int64_t sbt, int width, const int32_t* seq_lens,
                      const int32_t* query_start_loc, const int64_t* tree_mask, int n, int64_t tokens, int max_tokens,
                      int H, int KV, int D, int BS, float scale, int64_t max_len, void* out, int64_t so_t, int64_t so_h,
                      void* workspace, size_t workspace_bytes, void* stream) {
  if (n > 0 && !query_start_loc) return EX_ERR_ARG;
  return paged_rows(q, sq_t, sq_h, q_dtype, k_cache, v_cache, code, s_block, s_page, s_head, k_scale, v_scale, ss_block,
                    ss_head, num_blocks, block_table, sbt, width, seq_lens, query_start_loc, tree_mask, n, tokens,
                    max_tokens, H, KV, D, BS, scale, max_len, out, so_t, so_h, workspace, workspace_bytes,
                    (cudaStream_t)stream);
}

int ex_prompt_attention(const void* q, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_t, int64_t sk_h,
                        const void* v, int64_t sv_t, int64_t sv_h, int dtype, const int32_t* cu_q, const int32_t* cu_k,
                        int n, int64_t tokens, int64_t keys, int H, int KV, int D, float scale, void* out, int64_t so_t,
                        int64_t so_h, void* stream) {
  if (n < 0 || tokens < 0 || keys < 0 || tokens > INT32_MAX / 2 || keys > INT32_MAX / 2 || H <= 0 || KV <= 0 || H % KV != 0)
    return EX_ERR_ARG;
  if (!half_dtype(dtype)) return EX_ERR_DTYPE;
  if (!head_size_ok(D)) return EX_ERR_UNSUPPORTED;
  if (n == 0 || tokens == 0) return EX_OK;
  if (!q || !cu_q || !cu_k || !out || (keys > 0 && (!k || !v))) return EX_ERR_ARG;
  for (int64_t* s : {&sq_t, &so_t}) one_element(tokens, D, *s);
  for (int64_t* s : {&sk_t, &sv_t}) one_element(keys, D, *s);
  for (int64_t* s : {&sq_h, &so_h}) one_element(H, D, *s);
  for (int64_t* s : {&sk_h, &sv_h}) one_element(KV, D, *s);
  if (misaligned(q, 16) || misaligned(k, 16) || misaligned(v, 16) || misaligned(out, 16) || sq_t % 8 != 0 ||
      sq_h % 8 != 0 || sk_t % 8 != 0 || sk_h % 8 != 0 || sv_t % 8 != 0 || sv_h % 8 != 0 || so_t % 8 != 0 || so_h % 8 != 0)
    return EX_ERR_ALIGN;
  if (!(scale > 0.0f && scale * ex::PR_LOG2E < INFINITY)) return EX_ERR_ARG;
  if (!ex::device_is_sm100()) return EX_ERR_UNSUPPORTED;
  if (keys == 0) {  // nothing to map: any rows do, none of them is read
    k = v = q;
    sk_t = sv_t = sq_t;
    sk_h = sv_h = sq_h;
    KV = H;
  }
  CUtensorMap mq, mk, mv;
  if (!encode_packed_map(&mq, q, D, H, tokens, sq_h, sq_t) ||
      !encode_packed_map(&mk, k, D, KV, keys > 0 ? keys : tokens, sk_h, sk_t) ||
      !encode_packed_map(&mv, v, D, KV, keys > 0 ? keys : tokens, sv_h, sv_t))
    return EX_ERR_UNSUPPORTED;
  ex::PaArgs a = {};
  a.v = v; a.sv_t = sv_t; a.sv_h = sv_h;
  a.cu_q = cu_q; a.cu_k = cu_k; a.n = n; a.H = H; a.G = H / KV; a.tokens = tokens; a.keys = keys;
  a.scale_log2 = scale * ex::PR_LOG2E; a.out = out; a.so_t = so_t; a.so_h = so_h;
  cudaStream_t st = (cudaStream_t)stream;
  const bool f16 = dtype == EX_DTYPE_F16;
  if (D == 64) return f16 ? launch_prompt<64, true>(mq, mk, mv, a, st) : launch_prompt<64, false>(mq, mk, mv, a, st);
  if (D == 128) return f16 ? launch_prompt<128, true>(mq, mk, mv, a, st) : launch_prompt<128, false>(mq, mk, mv, a, st);
  return f16 ? launch_prompt<256, true>(mq, mk, mv, a, st) : launch_prompt<256, false>(mq, mk, mv, a, st);
}

int ex_cache_write_q8(const void* key, int64_t sk_t, int64_t sk_h, const void* value, int64_t sv_t, int64_t sv_h,
                      int dtype, int code, void* k_cache, void* v_cache, int64_t s_block, int64_t s_page, int64_t s_head,
                      float* k_scale, float* v_scale, int64_t ss_block, int64_t ss_head, int64_t num_blocks, int BS,
                      const int64_t* slots, int64_t tokens, int KV, int D, void* key_out, int64_t sko_t, int64_t sko_h,
                      void* value_out, int64_t svo_t, int64_t svo_h, void* stream) {
  if (tokens < 0) return EX_ERR_ARG;
  const int rc = check_cache(dtype, code, k_cache, v_cache, s_block, s_page, s_head, k_scale, v_scale, num_blocks, BS, KV, D);
  if (rc != EX_OK || tokens == 0) return rc;
  if (!key || !value || !slots || (!key_out) != (!value_out)) return EX_ERR_ARG;
  for (int64_t* s : {&sk_t, &sv_t, &sko_t, &svo_t}) one_element(tokens, D, *s);
  for (int64_t* s : {&sk_h, &sv_h, &sko_h, &svo_h}) one_element(KV, D, *s);
  if (misaligned(key, 16) || misaligned(value, 16) || misaligned(slots, 8) || sk_t % 8 != 0 || sk_h % 8 != 0 ||
      sv_t % 8 != 0 || sv_h % 8 != 0)
    return EX_ERR_ALIGN;
  if (key_out && (misaligned(key_out, 16) || misaligned(value_out, 16) || sko_t % 8 != 0 || sko_h % 8 != 0 ||
                  svo_t % 8 != 0 || svo_h % 8 != 0))
    return EX_ERR_ALIGN;
  if (tokens > INT32_MAX / 4 / KV) return EX_ERR_UNSUPPORTED;
  const ex::CacheView c = cache_view(k_cache, v_cache, s_block, s_page, s_head, k_scale, v_scale, ss_block, ss_head, num_blocks, BS);
  cudaStream_t st = (cudaStream_t)stream;
  const int f16 = dtype == EX_DTYPE_F16;
#define EX_CW(DD, CC)                                                                                                     \
  if (D == DD && code == CC)                                                                                              \
    return cuda_status((f16 ? launch_cache_write<DD, CC, __half> : launch_cache_write<DD, CC, __nv_bfloat16>)(            \
        key, value, sk_t, sk_h, sv_t, sv_h, c, slots, tokens, KV, key_out, value_out, sko_t, sko_h, svo_t, svo_h, st));
  EX_CW(64, ex::CODE_INT8)
  EX_CW(128, ex::CODE_INT8)
  EX_CW(256, ex::CODE_INT8)
  EX_CW(64, ex::CODE_E4M3)
  EX_CW(128, ex::CODE_E4M3)
  EX_CW(256, ex::CODE_E4M3)
#undef EX_CW
  return EX_ERR_UNSUPPORTED;
}

int ex_cache_read_q8(const void* k_cache, const void* v_cache, int code, int64_t s_block, int64_t s_page, int64_t s_head,
                     const float* k_scale, const float* v_scale, int64_t ss_block, int64_t ss_head, int64_t num_blocks,
                     int BS, const int32_t* block_table, int64_t sbt, int width, const int32_t* cu_seqlens, int n,
                     int64_t rows, int KV, int D, int dtype, void* key_out, int64_t sko_t, int64_t sko_h, void* value_out,
                     int64_t svo_t, int64_t svo_h, void* stream) {
  if (rows < 0 || n < 0 || width < 0) return EX_ERR_ARG;
  const int rc = check_cache(dtype, code, k_cache, v_cache, s_block, s_page, s_head, k_scale, v_scale, num_blocks, BS, KV, D);
  if (rc != EX_OK || rows == 0 || n == 0) return rc;
  if (!block_table || !cu_seqlens || !key_out || !value_out) return EX_ERR_ARG;
  for (int64_t* s : {&sko_t, &svo_t}) one_element(rows, D, *s);
  for (int64_t* s : {&sko_h, &svo_h}) one_element(KV, D, *s);
  if (misaligned(key_out, 16) || misaligned(value_out, 16) || sko_t % 8 != 0 || sko_h % 8 != 0 || svo_t % 8 != 0 || svo_h % 8 != 0)
    return EX_ERR_ALIGN;
  if (rows > INT32_MAX) return EX_ERR_UNSUPPORTED;
  const ex::CacheView c = cache_view(k_cache, v_cache, s_block, s_page, s_head, k_scale, v_scale, ss_block, ss_head, num_blocks, BS);
  cudaStream_t st = (cudaStream_t)stream;
  const int f16 = dtype == EX_DTYPE_F16;
#define EX_CR(DD, CC)                                                                                                  \
  if (D == DD && code == CC)                                                                                           \
    return cuda_status(launch_cache_read<DD, CC>(c, block_table, sbt, width, cu_seqlens, n, rows, KV, f16, key_out,    \
                                                 value_out, sko_t, sko_h, svo_t, svo_h, st));
  EX_CR(64, ex::CODE_INT8)
  EX_CR(128, ex::CODE_INT8)
  EX_CR(256, ex::CODE_INT8)
  EX_CR(64, ex::CODE_E4M3)
  EX_CR(128, ex::CODE_E4M3)
  EX_CR(256, ex::CODE_E4M3)
#undef EX_CR
  return EX_ERR_UNSUPPORTED;
}

}  // extern "C"
