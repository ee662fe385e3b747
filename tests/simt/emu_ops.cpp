// Host build of the serving operators' kernels (chunk attention, log
// probabilities, page copies) under the SIMT emulator, with a C entry point
// each for the CPU tests (ctypes).  Test infrastructure.
#include "simt.h"

#include <cuda.h>
#include <type_traits>

#define execute_mma execute_mma_i8
#include "simt_tcgen05.h"
#undef execute_mma

namespace simt {
// kind::f16 with A in tensor memory: D[m][n] (+)= sum_k A[m][k] B[n][k], K = 16
inline void execute_mma(const TensorOp& op) {
  Block* b = op.blk;
  const uint32_t id = op.idesc;
  if (((id >> 4) & 3u) != 1u) fail("tcgen05.mma kind::f16: accumulator type is not f32");
  if (((id >> 7) & 7u) || ((id >> 10) & 7u)) fail("tcgen05.mma kind::f16: operands are not f16");
  if ((id >> 15) & 1u) fail("tcgen05.mma: A in tensor memory is K-major");
  const bool mn_major = (id >> 16) & 1u;
  const int M = (int)((id >> 24) & 0x1Fu) << 4, N = (int)((id >> 17) & 0x3Fu) << 3;
  if (M != 128) fail("tcgen05.mma cta_group::1: only M = 128 is modelled");
  if (N < 16 || N > 256 || N % 16) fail("tcgen05.mma: N must be a multiple of 16 in [16, 256]");
  const uint32_t mode = (uint32_t)(op.bdesc >> 61) & 7u;  // swizzle: 2 128-byte, 4 64-byte rows
  if (mode != 2 && mode != 4) fail("tcgen05 matrix descriptor: swizzle mode not modelled");
  const uint32_t rb = mode == 2 ? 128 : 64;
  const SmemDesc B = decode_desc(op.bdesc & ~(7ull << 61));
  const uint32_t a_col = (uint32_t)op.adesc & 0xFFFFu, d_col = op.d_tmem & 0xFFFFu;
  if (((uint32_t)op.adesc >> 16) || (op.d_tmem >> 16)) fail("tcgen05.mma: M = 128 starts at lane 0");
  auto used = [&](uint32_t c0, uint32_t n) {
    if (c0 + n > 512) fail("tcgen05.mma past the last column");
    for (uint32_t u = c0 / 32; u <= (c0 + n - 1) / 32; ++u)
      if (!(b->tmem_used >> u & 1u)) fail("tcgen05.mma of tensor memory that is not allocated");
  };
  used(a_col, 8);
  used(d_col, (uint32_t)N);
  auto half_at = [](const uint8_t* p) {
    uint16_t u;
    memcpy(&u, p, 2);
    __half_raw r;
    r.x = u;
    return __half2float(__half(r));
  };
  std::vector<float> bv((size_t)N * 16);
  for (int n = 0; n < N; ++n)
    for (int k = 0; k < 16; ++k) {
      // 8 rows (K-major: N; MN-major: K) of rb bytes are SBO apart; N beyond a
      // row (MN-major) is LBO away; pieces move by the address bits above them
      const size_t row = mn_major ? k : n, col = (mn_major ? n : k) * 2;
      const size_t lin = B.start + row / 8 * B.sbo + row % 8 * rb + col / rb * B.lbo + col % rb;
      const size_t off = lin ^ ((lin >> 7 & (rb == 128 ? 7 : 3)) << 4);
      if (off + 2 > b->smem_bytes) fail("tcgen05.mma operand outside shared memory");
      bv[(size_t)n * 16 + k] = half_at(b->smem + off);
    }
  for (int m = 0; m < M; ++m) {
    float av[16];
    for (int k = 0; k < 16; ++k)
      av[k] = half_at(reinterpret_cast<const uint8_t*>(&b->tmem[(size_t)m * 512 + a_col]) + 2 * k);
    for (int n = 0; n < N; ++n) {
      float* cell = reinterpret_cast<float*>(&b->tmem[(size_t)m * 512 + d_col + n]);
      float s = op.accumulate ? *cell : 0.0f;
      for (int k = 0; k < 16; ++k) s += av[k] * bv[(size_t)n * 16 + k];
      *cell = s;
    }
  }
}
}  // namespace simt

inline unsigned __reduce_add_sync(unsigned mask, unsigned v) {
  uint64_t all[32], s = 0;
  simt::warp_exchange(mask, v, -1, "__reduce_add_sync", all);
  for (uint64_t x : all) s += x;
  return (unsigned)s;
}
inline int __ffs(unsigned v) { return __builtin_ffs((int)v); }
inline unsigned long long atomicMax(unsigned long long* p, unsigned long long v) {
  simt::yield();
  const unsigned long long o = *p;
  if (v > o) *p = v;
  simt::made_progress();
  return o;
}

#include "l3g.h"

#define L3G_PTX_HEADER "simt_l3g_ptx.h"
#include "l3g_kernels.cuh"

namespace l3g {
#include "simt_tc16.h"

#include "l3g_chunk_attn.cuh"

#include "l3g_logprobs.cuh"

#include "l3g_pages.cuh"
}  // namespace l3g

namespace {
std::string g_err;
template <typename F>
int guarded_call(F&& f) {
  try {
    f();
    return 0;
  } catch (const std::exception& e) {
    g_err = e.what();
    return -1;
  }
}
template <int HD, typename KT>
void run_chunk(const l3g::ChunkArgs& a, int grid) {
  simt::launch(dim3(grid), dim3(l3g::CHUNK_THREADS), l3g::chunk_smem_bytes(HD, (int)sizeof(KT)),
               [&] { l3g::k_chunk_attention<HD, KT>(a); });
  simt::launch(dim3(grid, l3g::CHUNK_BM / 8), dim3(256), 0, [&] { l3g::k_chunk_merge<HD>(a); },
               true);
}
}  // namespace

extern "C" {
const char* emu_error() { return g_err.c_str(); }
void emu_schedule(int randomize, unsigned long long seed, int max_copy_delay) {
  simt::rt().randomize = randomize != 0;
  simt::rt().rng.seed(seed);
  simt::rt().max_copy_delay = max_copy_delay;
}
void* emu_malloc(unsigned long long bytes) {
  void* p = nullptr;
  guarded_call([&] { p = simt::dmalloc(bytes); });
  return p;
}
void emu_free(void* p) { guarded_call([&] { simt::dfree(p); }); }

// Chunk attention on a grid of `grid` CTAs; every pointer from emu_malloc.
int emu_chunk_attention(const void* seqs, int n_seqs, int total_q, const float* q, long long ldq,
                        float* out, long long ldo, int layer, int heads, int hkv, int hd,
                        int kv_f16, float scale, int grid, int* err, int* where) {
  std::vector<void*> scratch;
  auto dm = [&](size_t bytes) {
    void* p = simt::dmalloc(bytes);
    scratch.push_back(p);
    return p;
  };
  const int rc = guarded_call([&] {
    l3g::ChunkArgs a{};
    a.seqs = static_cast<const l3g_chunk_seq*>(seqs);
    a.n_seqs = n_seqs;
    a.total_q = total_q;
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.layer = layer;
    a.hkv = hkv;
    a.group = heads / hkv;
    a.ginv = 65535 / a.group + 1;
    a.scale = (float)(scale * M_LOG2E);
    a.part_o = static_cast<float*>(dm((size_t)2 * grid * 128 * hd * 4));
    a.part_ml = static_cast<float*>(dm((size_t)2 * grid * 128 * 2 * 4));
    a.split = static_cast<int*>(dm((size_t)grid * 8 * 4));
    a.maps = static_cast<uint8_t*>(dm((size_t)grid * l3g::CHUNK_LOAD * 128));
    {
      const int es = kv_f16 ? 2 : 4;
      l3g::EmuMap m{nullptr, 2 * hd * es, l3g::chunk_row_bytes(hd, es), l3g::chunk_bn(es), es};
      memcpy(&a.map, &m, sizeof m);
    }
    a.res = static_cast<l3g::Result*>(dm(sizeof(l3g::Result)));
    a.wait_ns = 1ull << 60;
    if (hd == 32 && kv_f16) run_chunk<32, __half>(a, grid);
    else if (hd == 32) run_chunk<32, float>(a, grid);
    else if (hd == 64 && kv_f16) run_chunk<64, __half>(a, grid);
    else if (hd == 64) run_chunk<64, float>(a, grid);
    else if (kv_f16) run_chunk<128, __half>(a, grid);
    else run_chunk<128, float>(a, grid);
    *err = a.res->err;
    *where = a.res->where;
  });
  for (void* p : scratch) simt::dfree(p);
  return rc;
}

// Log probabilities of n rows as l3g_logprobs_run launches them, on at most
// max_grid CTAs; every pointer from emu_malloc (or null).
int emu_logprobs(const float* x, long long ld, int n, int vocab, const int* targets, float* logprob,
                 float* entropy, int* rank, int k, int* top_ids, float* top_lp, int vec, int max_grid,
                 int* err) {
  std::vector<void*> scratch;
  auto dm = [&](size_t bytes) {
    void* p = simt::dmalloc(bytes);
    scratch.push_back(p);
    return p;
  };
  const int rc = guarded_call([&] {
    l3g::LogprobArgs a{};
    a.x = x;
    a.ld = ld;
    a.n = n;
    a.vocab = vocab;
    a.k = k;
    a.slices = (vocab + l3g::LP_SLICE - 1) / l3g::LP_SLICE;
    a.targets = targets;
    a.logprob = logprob;
    a.entropy = entropy;
    a.rank = rank;
    a.top_ids = top_ids;
    a.top_lp = top_lp;
    a.res = static_cast<l3g::Result*>(dm(sizeof(l3g::Result)));
    a.wait_ns = 1ull << 60;
    a.part = static_cast<float4*>(dm((size_t)n * a.slices * sizeof(float4)));
    a.part_k = static_cast<uint64_t*>(dm((size_t)n * a.slices * std::max(k, 1) * 8));
    const dim3 grid(std::min(n * a.slices, max_grid));
    // (a grid of one is not sequential by itself: its arrays are static all the same)
    simt::seq_override() = true;
    simt::seq_grid() = grid;
    for (unsigned b = 0; b < grid.x; ++b) {
      simt::seq_bidx() = uint3{b, 0, 0};
      if (vec)
        simt::launch(dim3(1), dim3(l3g::LP_THREADS), l3g::LP_SMEM,
                     [&] { l3g::k_logprobs_part<true>(a); });
      else
        simt::launch(dim3(1), dim3(l3g::LP_THREADS), 0, [&] { l3g::k_logprobs_part<false>(a); });
    }
    simt::seq_grid() = dim3(n);
    for (int r = 0; r < n && a.slices > 1; ++r) {
      simt::seq_bidx() = uint3{(unsigned)r, 0, 0};
      simt::launch(dim3(1), dim3(l3g::LP_JOIN), 0, [&] { l3g::k_logprobs_join(a); });
    }
    *err = a.res->err;
  });
  simt::seq_override() = false;
  for (void* p : scratch) simt::dfree(p);
  return rc;
}

// Page copies as l3g_kv_copy_pages launches them, on at most max_rows grid rows.
int emu_copy_pages(const void* src_pool, int n_src, void* dst_pool, int n_dst, int row_bytes,
                   const int* src, const int* dst, const int* rows, int n, int* status, int max_rows) {
  return guarded_call([&] {
    simt::launch(dim3(l3g::COPY_SLICES, std::min(n, max_rows)), dim3(256), 0, [&] {
      l3g::k_copy_pages(static_cast<const uint8_t*>(src_pool), n_src, static_cast<uint8_t*>(dst_pool),
                        n_dst, row_bytes, src, dst, rows, n, status);
    });
  });
}
}
