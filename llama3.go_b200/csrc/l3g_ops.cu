// The serving operators: attention of token chunks over paged caches, log
// probabilities, page copies.
#include <cuda.h>

#include <type_traits>

#include "l3g_rt.h"

namespace l3g {
#include "l3g_tc16.cuh"

#include "l3g_chunk_attn.cuh"

#include "l3g_logprobs.cuh"

#include "l3g_pages.cuh"
}  // namespace l3g

// Makes `dev` current for a call and puts the caller's device back.
struct DeviceScope {
  int prev = -1;
  cudaError_t err = cudaSuccess;
  explicit DeviceScope(int dev) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != dev) err = cudaSetDevice(dev);
    if (prev == dev) prev = -1;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};
#define ON_DEVICE(dev)      \
  DeviceScope scope_(dev);  \
  CUDA_TRY(scope_.err)

static bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

// ---------------------------------------------------------------------------
// attention of token chunks
// ---------------------------------------------------------------------------
struct l3g_chunk_attn {
  int device = 0, nsm = 1;
  int heads = 0, hkv = 0, hd = 0, kv_f16 = 0;
  Result* d_res = nullptr;
  float* part_o = nullptr;   // pieces of row tiles that several CTAs share
  float* part_ml = nullptr;
  int* split = nullptr;
  uint8_t* maps = nullptr;   // the loaders' tensor maps
  CUtensorMap map;           // what they are made from
};

// The tensor map of a pool's rows in boxes of one panel: the base address is a
// placeholder that the kernel replaces, and rows are checked by page id there.
static int chunk_map(l3g_chunk_attn* h) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult found;
  CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000,
                                            cudaEnableDefault, &found));
  if (!fn || found != cudaDriverEntryPointSuccess)
    return l3g_fail(L3G_E_CUDA, "chunk attention: no cuTensorMapEncodeTiled in the driver");
  const int es = h->kv_f16 ? 2 : 4;
  const cuuint64_t dims[2] = {(cuuint64_t)2 * h->hd, 0x7fffffffull};
  const cuuint64_t strides[1] = {(cuuint64_t)2 * h->hd * es};
  const cuuint32_t box[2] = {(cuuint32_t)chunk_box_cols(h->hd, es), (cuuint32_t)chunk_bn(es)};
  const cuuint32_t step[2] = {1, 1};
  const CUresult r = reinterpret_cast<Encode>(fn)(
      &h->map, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2,
      h->part_o, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
      chunk_row_bytes(h->hd, es) == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return l3g_fail(L3G_E_CUDA, "chunk attention: tensor map, error %d", (int)r);
  return L3G_OK;
}

// Kernel attributes, once per device, with that device current.
static int chunk_setup() {
  static int rcs[64];
  static std::once_flag onces[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
    return l3g_fail(L3G_E_CUDA, "chunk attention set-up: no current device");
  int& rc = rcs[dev];
  std::call_once(onces[dev], [&rc] {
    cudaError_t e = cudaSuccess;
#define SETCA(HD, KT)                                                                       \
  if (e == cudaSuccess)                                                                    \
  e = cudaFuncSetAttribute(k_chunk_attention<HD, KT>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                           chunk_smem_bytes(HD, (int)sizeof(KT)))
    SETCA(32, float);
    SETCA(64, float);
    SETCA(128, float);
    SETCA(32, __half);
    SETCA(64, __half);
    SETCA(128, __half);
#undef SETCA
    rc = e == cudaSuccess ? L3G_OK
                          : l3g_fail(L3G_E_CUDA, "chunk attention attributes: %s",
                                     cudaGetErrorString(e));
  });
  return rc ? l3g_fail(L3G_E_CUDA, "chunk attention set-up failed on device %d", dev) : L3G_OK;
}

extern "C" void l3g_chunk_attn_free(l3g_chunk_attn* h) {
  if (!h) return;
  DeviceScope scope(h->device);
  void* d[] = {h->d_res, h->part_o, h->part_ml, h->split, h->maps};
  for (void* p : d)
    if (p) cudaFree(p);
  delete h;
}

extern "C" int l3g_chunk_attn_new(int32_t n_heads, int32_t n_heads_kv, int32_t head_dim,
                                  int32_t kv_dtype, int32_t device, l3g_chunk_attn** out) {
  if (!out) return l3g_fail(L3G_E_INVALID, "null argument");
  *out = nullptr;
  if (n_heads <= 0 || n_heads_kv <= 0 || n_heads % n_heads_kv || n_heads / n_heads_kv > MAXG ||
      n_heads_kv > 65535)
    return l3g_fail(L3G_E_INVALID, "chunk attention: %d query heads over %d kv heads", n_heads,
                    n_heads_kv);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return l3g_fail(L3G_E_INVALID, "chunk attention: head_dim %d", head_dim);
  if (kv_dtype != L3G_KV_F32 && kv_dtype != L3G_KV_F16)
    return l3g_fail(L3G_E_INVALID, "kv_dtype=%d", kv_dtype);
  int dev = device;
  if (dev < 0) CUDA_TRY(cudaGetDevice(&dev));
  ON_DEVICE(dev);
  if (int rc = chunk_setup()) return rc;
  auto* h = new l3g_chunk_attn();
  h->device = dev;
  h->nsm = sm_count(dev);
  h->heads = n_heads;
  h->hkv = n_heads_kv;
  h->hd = head_dim;
  h->kv_f16 = kv_dtype == L3G_KV_F16;
  cudaError_t e = cudaMalloc(&h->d_res, sizeof(Result));
  if (e == cudaSuccess) e = cudaMemset(h->d_res, 0, sizeof(Result));
  const size_t rows = (size_t)2 * h->nsm * CHUNK_BM;  // two pieces per CTA
  if (e == cudaSuccess) e = cudaMalloc(&h->part_o, rows * head_dim * 4);
  if (e == cudaSuccess) e = cudaMalloc(&h->part_ml, rows * 2 * 4);
  if (e == cudaSuccess) e = cudaMalloc(&h->split, (size_t)h->nsm * 8 * 4);
  if (e == cudaSuccess) e = cudaMalloc(&h->maps, (size_t)h->nsm * CHUNK_LOAD * 128);
  if (e != cudaSuccess) {
    l3g_chunk_attn_free(h);
    return l3g_fail(L3G_E_CUDA, "chunk attention: %s", cudaGetErrorString(e));
  }
  if (int rc = chunk_map(h)) {
    l3g_chunk_attn_free(h);
    return rc;
  }
  *out = h;
  return L3G_OK;
}

template <int HD, typename KT>
static cudaError_t launch_chunk(const l3g_chunk_attn* h, const ChunkArgs& a, cudaStream_t st) {
  k_chunk_attention<HD, KT>
      <<<h->nsm, CHUNK_THREADS, chunk_smem_bytes(HD, (int)sizeof(KT)), st>>>(a);
  if (const cudaError_t e = cudaGetLastError()) return e;
  cudaLaunchAttribute at{};  // launched early: it waits for the pieces itself
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(h->nsm, CHUNK_BM / 8);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_chunk_merge<HD>, a);
}

extern "C" int l3g_chunk_attn_run(l3g_chunk_attn* h, const l3g_chunk_seq* seqs, int32_t n_seqs,
                                  int32_t total_q, const float* q, int64_t ldq, float* out,
                                  int64_t ldo, int32_t layer, float scale, void* stream) {
  if (!h) return l3g_fail(L3G_E_INVALID, "null argument");
  if (n_seqs < 0 || n_seqs > L3G_CHUNK_SEQS_MAX)
    return l3g_fail(L3G_E_INVALID, "n_seqs=%d outside [0, %d]", n_seqs, L3G_CHUNK_SEQS_MAX);
  if (total_q < 0 || layer < 0)
    return l3g_fail(L3G_E_INVALID, "total_q=%d, layer=%d", total_q, layer);
  if (n_seqs == 0 || total_q == 0) return L3G_OK;
  if (!seqs || !q || !out) return l3g_fail(L3G_E_INVALID, "null argument");
  const int64_t width = (int64_t)h->heads * h->hd;
  if (ldq < width || ldo < width || ldq % 4 || ldo % 4)
    return l3g_fail(L3G_E_INVALID, "row strides %lld and %lld: multiples of 4, at least %lld",
                    (long long)ldq, (long long)ldo, (long long)width);
  if (misaligned(q, 16) || misaligned(out, 16) || misaligned(seqs, 8))
    return l3g_fail(L3G_E_INVALID, "q and out must be 16-byte aligned, seqs 8-byte");
  if (std::isnan(scale) || std::isinf(scale)) return l3g_fail(L3G_E_INVALID, "scale not finite");
  ON_DEVICE(h->device);
  ChunkArgs a{};
  a.seqs = seqs;
  a.n_seqs = n_seqs;
  a.total_q = total_q;
  a.q = q;
  a.ldq = ldq;
  a.out = out;
  a.ldo = ldo;
  a.layer = layer;
  a.hkv = h->hkv;
  a.group = h->heads / h->hkv;
  a.ginv = 65535 / a.group + 1;
  a.scale = (float)((scale > 0.0f ? (double)scale : 1.0 / sqrt((double)h->hd)) * M_LOG2E);
  a.res = h->d_res;
  a.part_o = h->part_o;
  a.part_ml = h->part_ml;
  a.split = h->split;
  a.maps = h->maps;
  a.map = h->map;
  a.wait_ns = WAIT_TIMEOUT_NS;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (h->kv_f16)
    e = h->hd == 32 ? launch_chunk<32, __half>(h, a, st)
                    : h->hd == 64 ? launch_chunk<64, __half>(h, a, st)
                                  : launch_chunk<128, __half>(h, a, st);
  else
    e = h->hd == 32 ? launch_chunk<32, float>(h, a, st)
                    : h->hd == 64 ? launch_chunk<64, float>(h, a, st)
                                  : launch_chunk<128, float>(h, a, st);
  CUDA_TRY(e);
  return L3G_OK;
}

extern "C" int l3g_chunk_attn_status(l3g_chunk_attn* h, int32_t* err, int32_t* where) {
  if (!h || !err || !where) return l3g_fail(L3G_E_INVALID, "null argument");
  ON_DEVICE(h->device);
  CUDA_TRY(cudaDeviceSynchronize());
  Result r{};
  CUDA_TRY(cudaMemcpy(&r, h->d_res, sizeof r, cudaMemcpyDeviceToHost));
  CUDA_TRY(cudaMemset(h->d_res, 0, sizeof(Result)));
  *err = r.err;
  *where = r.where;
  return L3G_OK;
}

// ---------------------------------------------------------------------------
// log probabilities
// ---------------------------------------------------------------------------
struct l3g_logprobs {
  int device = 0, nsm = 1;
  int max_rows = 0, vocab = 0;
  float4* part = nullptr;      // the slices' sums
  uint64_t* part_k = nullptr;  // and top keys
  Result* d_res = nullptr;     // device error word of the kernel's bounded waits
};

extern "C" void l3g_logprobs_free(l3g_logprobs* h) {
  if (!h) return;
  DeviceScope scope(h->device);
  if (h->part) cudaFree(h->part);
  if (h->part_k) cudaFree(h->part_k);
  if (h->d_res) cudaFree(h->d_res);
  delete h;
}

// Kernel attributes, once per device, with that device current.
static int logprob_setup() {
  static int rcs[64];
  static std::once_flag onces[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
    return l3g_fail(L3G_E_CUDA, "log probabilities set-up: no current device");
  int& rc = rcs[dev];
  std::call_once(onces[dev], [&rc] {
    const cudaError_t e = cudaFuncSetAttribute(
        k_logprobs_part<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, LP_SMEM);
    rc = e == cudaSuccess ? L3G_OK
                          : l3g_fail(L3G_E_CUDA, "log probabilities attributes: %s",
                                     cudaGetErrorString(e));
  });
  return rc ? l3g_fail(L3G_E_CUDA, "log probabilities set-up failed on device %d", dev) : L3G_OK;
}

extern "C" int l3g_logprobs_new(int32_t max_rows, int32_t vocab, int32_t device,
                                l3g_logprobs** out) {
  if (!out) return l3g_fail(L3G_E_INVALID, "null argument");
  *out = nullptr;
  if (max_rows <= 0 || max_rows > (1 << 20) || vocab <= 0 || vocab > (1 << 24))
    return l3g_fail(L3G_E_INVALID, "log probabilities of %d rows of %d", max_rows, vocab);
  int dev = device;
  if (dev < 0) CUDA_TRY(cudaGetDevice(&dev));
  ON_DEVICE(dev);
  if (int rc = logprob_setup()) return rc;
  auto* h = new l3g_logprobs();
  h->device = dev;
  h->nsm = sm_count(dev);
  h->max_rows = max_rows;
  h->vocab = vocab;
  const size_t parts = (size_t)max_rows * ((vocab + LP_SLICE - 1) / LP_SLICE);
  cudaError_t e = cudaMalloc(&h->part, parts * sizeof(float4));
  if (e == cudaSuccess)
    e = cudaMalloc(&h->part_k, parts * std::min(MAX_TOPK, vocab) * sizeof(uint64_t));
  if (e == cudaSuccess) e = cudaMalloc(&h->d_res, sizeof(Result));
  if (e == cudaSuccess) e = cudaMemset(h->d_res, 0, sizeof(Result));
  if (e != cudaSuccess) {
    l3g_logprobs_free(h);
    return l3g_fail(L3G_E_CUDA, "log probabilities: %s", cudaGetErrorString(e));
  }
  *out = h;
  return L3G_OK;
}

extern "C" int l3g_logprobs_run(l3g_logprobs* h, const float* logits, int64_t ld, int32_t n,
                                const int32_t* targets, float* logprob, float* entropy,
                                int32_t* rank, int32_t top_k, int32_t* top_ids,
                                float* top_logprobs, void* stream) {
  if (!h) return l3g_fail(L3G_E_INVALID, "null argument");
  if (n < 0 || n > h->max_rows)
    return l3g_fail(L3G_E_INVALID, "n=%d outside [0, %d]", n, h->max_rows);
  if (top_k < 0 || top_k > MAX_TOPK || top_k > h->vocab)
    return l3g_fail(L3G_E_INVALID, "top_k=%d outside [0, %d]", top_k,
                    std::min(MAX_TOPK, h->vocab));
  if (ld < h->vocab)
    return l3g_fail(L3G_E_INVALID, "row stride %lld below the vocabulary %d", (long long)ld,
                    h->vocab);
  if (n == 0) return L3G_OK;
  if (!logits || (!targets && (logprob || rank)))
    return l3g_fail(L3G_E_INVALID, "null argument");
  const void* ps[] = {logits, targets, logprob, entropy, rank, top_ids, top_logprobs};
  for (const void* p : ps)
    if (misaligned(p, 4)) return l3g_fail(L3G_E_INVALID, "pointers must be 4-byte aligned");
  if (!top_ids && !top_logprobs) top_k = 0;
  ON_DEVICE(h->device);
  LogprobArgs a{};
  a.x = logits;
  a.ld = ld;
  a.n = n;
  a.vocab = h->vocab;
  a.k = top_k;
  a.targets = targets;
  a.logprob = logprob;
  a.entropy = entropy;
  a.rank = rank;
  a.top_ids = top_ids;
  a.top_lp = top_logprobs;
  a.slices = (h->vocab + LP_SLICE - 1) / LP_SLICE;
  a.part = h->part;
  a.part_k = h->part_k;
  const bool vec = !misaligned(logits, 16) && ld % 4 == 0;
  const cudaStream_t st = (cudaStream_t)stream;
  a.res = h->d_res;
  a.wait_ns = WAIT_TIMEOUT_NS;
  const int grid = (int)std::min<long long>((long long)n * a.slices, 3LL * h->nsm);
  if (vec) k_logprobs_part<true><<<grid, LP_THREADS, LP_SMEM, st>>>(a);
  else k_logprobs_part<false><<<grid, LP_THREADS, 0, st>>>(a);
  CUDA_TRY(cudaGetLastError());
  if (a.slices > 1) {  // launched early: it waits for the slices itself
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(n);
    cfg.blockDim = dim3(LP_JOIN);
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, k_logprobs_join, a));
  }
  return L3G_OK;
}

// Synchronizes the device; the error word of the kernels' bounded waits.
extern "C" int l3g_logprobs_status(l3g_logprobs* h, int32_t* err, int32_t* where) {
  if (!h || !err || !where) return l3g_fail(L3G_E_INVALID, "null argument");
  ON_DEVICE(h->device);
  CUDA_TRY(cudaDeviceSynchronize());
  Result r{};
  CUDA_TRY(cudaMemcpy(&r, h->d_res, sizeof r, cudaMemcpyDeviceToHost));
  CUDA_TRY(cudaMemset(h->d_res, 0, sizeof(Result)));
  *err = r.err;
  *where = r.where;
  return L3G_OK;
}

Result* chunk_attn_word(l3g_chunk_attn* h) { return h->d_res; }
Result* logprobs_word(l3g_logprobs* h) { return h->d_res; }

// ---------------------------------------------------------------------------
// page copies
// ---------------------------------------------------------------------------
extern "C" int l3g_kv_copy_pages(const void* src_pool, int32_t n_src, void* dst_pool,
                                 int32_t n_dst, int32_t row_bytes, const int32_t* src,
                                 const int32_t* dst, const int32_t* rows, int32_t n,
                                 int32_t* status, void* stream) {
  if (n < 0 || n_src < 0 || n_dst < 0)
    return l3g_fail(L3G_E_INVALID, "n=%d, pools of %d and %d pages", n, n_src, n_dst);
  if (row_bytes <= 0 || row_bytes % 16 || row_bytes > 65536)
    return l3g_fail(L3G_E_INVALID, "rows of %d bytes: a multiple of 16, at most 65536", row_bytes);
  if (n == 0) return L3G_OK;
  if (!src_pool || !dst_pool || !src || !dst) return l3g_fail(L3G_E_INVALID, "null argument");
  if (misaligned(src_pool, 16) || misaligned(dst_pool, 16) || misaligned(src, 4) ||
      misaligned(dst, 4) || misaligned(rows, 4) || misaligned(status, 4))
    return l3g_fail(L3G_E_INVALID, "pools must be 16-byte aligned, arrays 4-byte");
  k_copy_pages<<<dim3(COPY_SLICES, std::min(n, 65535)), 256, 0, (cudaStream_t)stream>>>(
      static_cast<const uint8_t*>(src_pool), n_src, static_cast<uint8_t*>(dst_pool), n_dst,
      row_bytes, src, dst, rows, n, status);
  CUDA_TRY(cudaGetLastError());
  return L3G_OK;
}
