// Attention of ragged chunks of new tokens over paged caches (included by
// l3g_ops.cu inside namespace l3g, after l3g_tc16.cuh).
//
// For every token i of a sequence and query head h (kv head h / G):
//   s_j = scale q.K_j,  j < kv_len - n_q + i + 1;  out = sum_j p_j V_j / sum_j p_j,
//   p_j = 2^(s_j log2 e - m), m the running maximum.
// Rows: the G query heads of a kv head times 128 / G consecutive tokens make
// one row tile of 128 rows (row r: token r / G, head r % G), which is the M of
// both products; the cache is taken in tiles of CHUNK_BN keys.
//
// Precision.  q, out and the statistics are fp32; the products run on the f16
// tensor cores.  An fp32 operand x goes in as two f16 terms, hi = f16(x) and
// lo = f16(x - hi), after scaling by a power of two (exact, undone in fp32), so
// it keeps 22 bits: q scaled per row, the weights p by 2^13, the K and V tiles
// of an f32 cache per tile; f16 caches go in as they are.  An f16 cache takes
// two products per tile (hi K, lo K), an f32 cache three (the lo lo term is
// below 2^-22).  The accumulators of one tile are fp32 in tensor memory; the
// sum over tiles is fp32 in registers, rounded to nearest, because the tensor
// core's own accumulation truncates and a long cache would add that up.
#pragma once

constexpr int CHUNK_BM = 128;       // rows per tile: lanes of tensor memory
constexpr int CHUNK_BN = 64;        // keys per tile; divides KV_PAGE
constexpr int CHUNK_SOFT = 8;       // softmax warps: two groups of four
constexpr int CHUNK_LOAD = 7;       // loader warps
constexpr int CHUNK_THREADS = 32 * (CHUNK_SOFT + CHUNK_LOAD + 1);
constexpr int CHUNK_MIN_TILES = 4;  // tiles a CTA takes at least
// tensor-memory columns: scores / weights of the two groups, q hi and lo, the
// two groups' tile outputs
constexpr uint32_t CHUNK_T_S = 0, CHUNK_T_Q = 128, CHUNK_T_O = 256, CHUNK_T_COLS = 512;

struct ChunkArgs {
  const l3g_chunk_seq* seqs;
  int n_seqs, total_q;
  const float* q;
  long long ldq;
  float* out;
  long long ldo;
  int layer, hkv, group;
  float scale;       // of the scores, times log2 e
  float* part_o;     // [2 * grid][128][HD] outputs of split row tiles
  float* part_ml;    // [2 * grid][128][2] their maxima and sums
  int* split;        // [grid][8] the split row tile that ends in a CTA
  Result* res;
  unsigned long long wait_ns;
};

struct ChunkSmem {
  uint64_t full[12], empty[12];  // K / V slots
  uint64_t s_full[2], p_full[2], o_full[2], o_free[2];
  uint64_t q_ready, xchg, lmax, drain;
  uint32_t tmem_base;
  int abort_flag;
  int n_tiles_lo, pad;
  long long begin, end;          // the CTA's range of the linear tile order
  long long unit0;               // first tile of the unit that holds `begin`
  int s0, kvh0, rt0, per;
  int bad[16];                   // segment + 1 whose pages are out of bounds
  float scale[32];               // f32 caches: 2^e of the items' tiles, item & 31
  float max[2][8];               // loader warps' maxima
  float ml[2][CHUNK_BM][2];      // the groups' statistics
  long long pre[L3G_CHUNK_SEQS_MAX + 1];  // tiles before each sequence
};
constexpr int CHUNK_HEAD = 11264;
static_assert(sizeof(ChunkSmem) <= CHUNK_HEAD, "chunk attention smem head");
constexpr int CHUNK_TBUF = 32 * 33 * 4;  // a softmax warp's transposition buffer
__host__ __device__ constexpr int chunk_slot_bytes(int hd, int es) {
  return CHUNK_BN * hd * es;  // f16: one operand tile; f32: its hi and lo tiles
}
__host__ __device__ constexpr int chunk_slots(int hd, int es) {
  return (180 * 1024) / chunk_slot_bytes(hd, es) < 12 ? (180 * 1024) / chunk_slot_bytes(hd, es)
                                                       : 12;
}
__host__ __device__ constexpr int chunk_smem_bytes(int hd, int es) {
  return CHUNK_HEAD + CHUNK_SOFT * CHUNK_TBUF + chunk_slots(hd, es) * chunk_slot_bytes(hd, es);
}

// Whether a descriptor stays inside its bounds (its pages are checked where
// they are read).
__device__ __forceinline__ bool chunk_seq_ok(const l3g_chunk_seq& s, int total_q) {
  return s.pool && s.pages && s.pps >= 0 && s.q0 >= 0 && s.n_q >= 0 && s.n_q <= total_q &&
         s.q0 <= total_q - s.n_q && s.kv_len >= 0 &&
         (long long)s.kv_len <= (long long)s.pps * KV_PAGE;
}
// Key tiles of row tile rt (at least one: a row that sees nothing is written)
__device__ __forceinline__ int chunk_tiles(const l3g_chunk_seq& s, int tt, int rt) {
  const long long end = (long long)(rt + 1) * tt;
  const long long see = (long long)s.kv_len - s.n_q + (end < s.n_q ? end : s.n_q);
  return see <= CHUNK_BN ? 1 : (int)((see + CHUNK_BN - 1) / CHUNK_BN);
}

// The CTAs share the linear order (sequence, kv head, row tile, key tile) in
// equal ranges; a row tile whose keys several CTAs hold is joined by
// k_chunk_merge.  A cursor walks a CTA's range in segments, each the key tiles
// [j0, j1) of one row tile.
struct ChunkCursor {
  long long pos, unit;  // next tile, first tile of its row tile
  int s, kvh, rt, seg;
  l3g_chunk_seq q;      // the sequence's descriptor
  int nk, j0, j1;
};
__device__ __forceinline__ void chunk_open(const ChunkArgs& a, ChunkCursor& c, long long end) {
  c.nk = chunk_tiles(c.q, CHUNK_BM / a.group, c.rt);
  c.j0 = (int)(c.pos - c.unit);
  c.j1 = (int)(end - c.unit < c.nk ? end - c.unit : c.nk);
}
__device__ __forceinline__ bool chunk_first(const ChunkArgs& a, const ChunkSmem* sh,
                                            ChunkCursor& c) {
  if (sh->begin >= sh->end) return false;
  c.pos = sh->begin;
  c.unit = sh->unit0;
  c.s = sh->s0;
  c.kvh = sh->kvh0;
  c.rt = sh->rt0;
  c.seg = 0;
  c.q = a.seqs[c.s];
  chunk_open(a, c, sh->end);
  return true;
}
__device__ __forceinline__ bool chunk_next(const ChunkArgs& a, const ChunkSmem* sh,
                                           ChunkCursor& c) {
  c.pos = c.unit + c.j1;
  if (c.pos >= sh->end) return false;
  c.unit = c.pos;  // a segment that ends before `end` ends its row tile
  ++c.seg;
  const int tt = CHUNK_BM / a.group;
  if (++c.rt >= (c.q.n_q + tt - 1) / tt) {
    c.rt = 0;
    if (++c.kvh >= a.hkv) {
      c.kvh = 0;
      do ++c.s;
      while (sh->pre[c.s + 1] == sh->pre[c.s]);
      c.q = a.seqs[c.s];
    }
  }
  chunk_open(a, c, sh->end);
  return true;
}

// Warp 0: the tiles of every sequence, then this CTA's range and where it starts.
__device__ __forceinline__ void chunk_plan(const ChunkArgs& a, ChunkSmem* sh, int lane) {
  const int tt = CHUNK_BM / a.group;
  long long sum = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    const int s = s0 + lane;
    long long n = 0;
    if (s < a.n_seqs) {
      const l3g_chunk_seq q = a.seqs[s];
      if (chunk_seq_ok(q, a.total_q)) {
        for (int rt = 0; rt < (q.n_q + tt - 1) / tt; ++rt) n += chunk_tiles(q, tt, rt);
        n *= a.hkv;
      } else if (blockIdx.x == 0) {
        report(a.res, ERR_SEQ, s);
      }
    }
    long long inc = n;  // inclusive scan
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (s < a.n_seqs) sh->pre[s] = sum + inc - n;
    sum += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) sh->pre[a.n_seqs] = sum;
  __syncwarp();
  if (lane == 0) {
    long long ctas = (sum + CHUNK_MIN_TILES - 1) / CHUNK_MIN_TILES;
    if (ctas > (long long)gridDim.x) ctas = gridDim.x;
    sh->begin = sh->end = 0;
    if ((long long)blockIdx.x < ctas) {
      sh->begin = sum * blockIdx.x / ctas;
      sh->end = sum * (blockIdx.x + 1) / ctas;
      int lo = 0, hi = a.n_seqs - 1;  // the last sequence that starts at or before it
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (sh->pre[mid] <= sh->begin) lo = mid;
        else hi = mid - 1;
      }
      const l3g_chunk_seq q = a.seqs[lo];
      long long unit = sh->pre[lo];
      const long long per = (sh->pre[lo + 1] - unit) / a.hkv;
      const int kvh = (int)((sh->begin - unit) / per);
      unit += per * kvh;
      int rt = 0;
      for (;; ++rt) {
        const int nk = chunk_tiles(q, tt, rt);
        if (sh->begin < unit + nk) break;
        unit += nk;
      }
      sh->s0 = lo;
      sh->kvh0 = kvh;
      sh->rt0 = rt;
      sh->unit0 = unit;
    }
  }
}

// The CTA whose range holds linear tile t.
__device__ __forceinline__ int chunk_owner(long long t, long long sum, int ctas) {
  int c = (int)(t * ctas / sum);
  while (c + 1 < ctas && sum * (c + 1) / ctas <= t) ++c;
  while (c > 0 && sum * c / ctas > t) --c;
  return c;
}

// o[d] = sum_j p_j V_j[d0 + d], d < 32, over the n keys of `rows` that a row
// sees, in fp32 from the cache itself: for a tile whose unseen keys hold a NaN
// or an infinity, which the product would multiply by zero.  o is shared
// memory of this thread's own; small loops, as it hardly ever runs.
template <int HD, typename KT>
__device__ __forceinline__ void chunk_row_slow(const KT* rows, int n, const float* q, float scale,
                                               float m, int d0, float* o) {
#pragma unroll 1
  for (int d = 0; d < 32; ++d) o[d] = 0.0f;
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const KT* k = rows + (size_t)j * 2 * HD;
    float s = 0.0f;
#pragma unroll 1
    for (int d = 0; d < HD; ++d) s = fmaf(q[d], (float)k[d], s);
    const float p = ex2(fmaf(s, scale, 13.0f - m));
#pragma unroll 1
    for (int d = 0; d < 32; ++d) o[d] = fmaf(p, (float)k[HD + d0 + d], o[d]);
  }
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
// 2^e as a float, e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// the exponent of the largest magnitude m, limited so that pow2i takes the
// scale factors that come from it; NaN and infinity count as the largest
__device__ __forceinline__ int exp_of(float m) {
  const int e = (__float_as_int(m) >> 23 & 255) - 127;
  return e < -100 ? -100 : e > 127 ? 127 : e;
}

// Roles: softmax groups 0 and 1 (warps 0-3 and 4-7; thread = row), taking the
// segment's key tiles in turn, each with statistics and an output of its own,
// joined at the segment's end; loader warps 8-14, which bring K and V tiles
// into a ring of shared-memory slots in the order the products use them
// (K0 K1 V0 K2 V1 ...); warp 15, whose lane 0 issues the products:
//   S = q K^T   A = q from tensor memory, B = K tile  [key][dim], K-major
//   O = p V     A = p from tensor memory (over S), B = V tile [key][dim], MN-major
// Both tiles sit as 16-byte pieces (8 dims of a key): piece c of key k at
// (c * BN + k) * 16, the canonical layout without swizzle either way.
template <int HD, typename KT>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
    k_chunk_attention(const __grid_constant__ ChunkArgs a) {
  constexpr int ES = (int)sizeof(KT);
  constexpr int BN = CHUNK_BN;
  constexpr int NS = chunk_slots(HD, ES);
  constexpr int SLOT = chunk_slot_bytes(HD, ES);
  constexpr int PARTS = ES == 4 ? 2 : 1;   // operand tiles per slot: hi (, lo)
  constexpr int PART = BN * HD * 2;
  L3G_DYNAMIC_SMEM(smem);
  ChunkSmem* sh = reinterpret_cast<ChunkSmem*>(smem);
  float* tbuf = reinterpret_cast<float*>(smem + CHUNK_HEAD);
  uint8_t* ring = smem + CHUNK_HEAD + CHUNK_SOFT * CHUNK_TBUF;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tt = CHUNK_BM / a.group;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh->full[i], CHUNK_LOAD);
      mbar_init(&sh->empty[i], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh->s_full[w], 1);
      mbar_init(&sh->p_full[w], 4);
      mbar_init(&sh->o_full[w], 1);
      mbar_init(&sh->o_free[w], 4);
    }
    mbar_init(&sh->q_ready, CHUNK_SOFT);
    mbar_init(&sh->xchg, CHUNK_SOFT);
    mbar_init(&sh->lmax, CHUNK_LOAD);
    mbar_init(&sh->drain, 1);
    sh->abort_flag = 0;
    for (int i = 0; i < 16; ++i) sh->bad[i] = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    __syncwarp();
    chunk_plan(a, sh, lane);
  }
  if (warp == 15) tmem_alloc(&sh->tmem_base, CHUNK_T_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  ChunkCursor c;
  bool more = chunk_first(a, sh, c);

  // two warpgroups give 64 of their 128 registers a thread to the other two
  if (warp >= CHUNK_SOFT) {
  regs_dec<64>();
  if (warp < CHUNK_SOFT + CHUNK_LOAD) {
    // ---- loaders ----------------------------------------------------------
    const int lw = warp - CHUNK_SOFT;
    const int kl = lane & 7, cl = lane >> 3;  // key and piece of the lane in an 8 x 4 patch
    constexpr int PATCHES = (BN / 8) * (HD / 32);
    constexpr int PER = (PATCHES + CHUNK_LOAD - 1) / CHUNK_LOAD;
    int it = 0;       // slots filled so far
    int pending = 0;  // f16: slots copied but not yet handed over
    bool ok = true;
    auto hand_over = [&](int slot) {
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->full[slot]);
    };
    for (; more && ok; more = chunk_next(a, sh, c)) {
      const int n = c.j1 - c.j0;
      const int* pages = c.q.pages + ((size_t)a.layer * a.hkv + c.kvh) * c.q.pps;
      for (int i = 0; i < 2 * n; ++i, ++it) {
        const bool is_v = i == 2 * n - 1 || (i > 0 && i % 2 == 0);
        const int j = c.j0 + (i == 2 * n - 1 ? n - 1 : is_v ? i / 2 - 1 : (i + 1) / 2);
        const int slot = it % NS;
        if (it >= NS) {
          ok = __all_sync(0xffffffffu, mbar_wait(&sh->empty[slot], (it / NS - 1) & 1,
                                                 &sh->abort_flag, a.res, 40, a.wait_ns));
          if (!ok) break;
        }
        const int kb = j * BN;
        int cnt = c.q.kv_len - kb;  // keys of the tile that exist
        cnt = cnt < 0 ? 0 : cnt > BN ? BN : cnt;
        int page = 0;
        if (cnt > 0) {
          page = pages[kb / KV_PAGE];
          if (page < 0 || page >= c.q.n_pages) {
            if (lane == 0) {
              report(a.res, ERR_PAGE, page);
              *(volatile int*)&sh->bad[c.seg & 15] = c.seg + 1;
            }
            page = 0;
            cnt = 0;
          }
        }
        const KT* src = reinterpret_cast<const KT*>(c.q.pool) +
                        ((size_t)page * KV_PAGE + (kb & (KV_PAGE - 1))) * 2 * HD +
                        (is_v ? HD : 0);
        uint8_t* dst = ring + (size_t)slot * SLOT;
        if constexpr (ES == 2) {
          for (int p = lw; p < PATCHES; p += CHUNK_LOAD) {
            const int k = (p % (BN / 8)) * 8 + kl, pc = (p / (BN / 8)) * 4 + cl;
            cp_async16(dst + (pc * BN + k) * 16,
                       k < cnt ? (const void*)(src + (size_t)k * 2 * HD + pc * 8) : c.q.pool,
                       k < cnt ? 16u : 0u);
          }
          cp_async_commit();
          if (pending == 3) {
            cp_async_wait<3>();
            hand_over((it - 3) % NS);
          } else {
            ++pending;
          }
        } else {
          float4 v[PER][2];
          float m = 0.0f;
#pragma unroll
          for (int r = 0; r < PER; ++r) {
            const int p = lw + r * CHUNK_LOAD;
            const int k = (p % (BN / 8)) * 8 + kl, pc = (p / (BN / 8)) * 4 + cl;
            v[r][0] = v[r][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p < PATCHES && k < cnt) {
              const float4* g = reinterpret_cast<const float4*>(src + (size_t)k * 2 * HD + pc * 8);
              v[r][0] = g[0];
              v[r][1] = g[1];
            }
          }
#pragma unroll
          for (int r = 0; r < PER; ++r) {
            const float* f = reinterpret_cast<const float*>(v[r]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = fabsf(f[e]);
              if (x <= 3.4028235e38f) m = fmaxf(m, x);
            }
          }
          m = warp_max(m);
          if (lane == 0) {
            sh->max[it & 1][lw] = m;
            mbar_arrive(&sh->lmax);
          }
          ok = __all_sync(0xffffffffu, mbar_wait(&sh->lmax, it & 1, &sh->abort_flag, a.res, 41,
                                                 a.wait_ns));
          if (!ok) break;
#pragma unroll
          for (int w = 0; w < CHUNK_LOAD; ++w) m = fmaxf(m, sh->max[it & 1][w]);
          const int e2 = exp_of(m);  // the tile's largest value lands in [2^14, 2^15)
          const float up = pow2i(14 - e2 > 127 ? 127 : 14 - e2);
          if (lane == 0 && lw == 0) sh->scale[it & 31] = 1.0f / up;
#pragma unroll
          for (int r = 0; r < PER; ++r) {
            const int p = lw + r * CHUNK_LOAD;
            if (p >= PATCHES) break;
            const int k = (p % (BN / 8)) * 8 + kl, pc = (p / (BN / 8)) * 4 + cl;
            const float* f = reinterpret_cast<const float*>(v[r]);
            uint4 hi, lo;
            uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
            uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = f[2 * e] * up, y = f[2 * e + 1] * up;
              h[e] = pack_h2(x, y);
              const float2 b = unpack_h2(h[e]);
              l[e] = pack_h2(x - b.x, y - b.y);
            }
            *reinterpret_cast<uint4*>(dst + (pc * BN + k) * 16) = hi;
            *reinterpret_cast<uint4*>(dst + PART + (pc * BN + k) * 16) = lo;
          }
          hand_over(slot);
        }
      }
    }
    if constexpr (ES == 2) {
      cp_async_wait<0>();
      for (; ok && pending > 0; --pending) hand_over((it - pending) % NS);
    }
  } else {
    // ---- product issuer -----------------------------------------------------
    if (lane == 0) {
      // f16 operands, f32 accumulators (bits 4-5 = 1), M >> 4 at 24, N >> 3 at
      // 17; B of the second product MN-major (bit 16)
      constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | (8u << 24);
      constexpr uint32_t IDESC_O =
          (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
      int it = 0;
      int cnt[2] = {0, 0};   // tiles of each group issued to S, over all segments
      int pcnt[2] = {0, 0};  // ... to O
      bool ok = true, any = false;
      auto wait = [&](uint64_t* b, int phase, int site) {
        return mbar_wait(b, phase & 1, &sh->abort_flag, a.res, site, a.wait_ns);
      };
      for (; more && ok; more = chunk_next(a, sh, c)) {
        const int n = c.j1 - c.j0;
        if (!wait(&sh->q_ready, c.seg, 42)) break;
        tc_fence_after();
        for (int j = 0; j <= n && ok; ++j) {
          if (j < n) {
            const int w = j & 1, slot = it % NS;
            ok = wait(&sh->full[slot], it / NS, 43);
            // the weights of the group's previous tile lie over S until its
            // second product is complete
            if (ok && cnt[w] > 0) ok = wait(&sh->o_full[w], cnt[w] - 1, 44);
            if (!ok) break;
            tc_fence_after();
            const uint32_t b0 = smem_u32(ring + (size_t)slot * SLOT);
            const uint32_t d = tmem + CHUNK_T_S + w * BN;
            bool acc = false;
            // small terms first: q_lo K_hi, (q_hi K_lo,) q_hi K_hi
#pragma unroll
            for (int t = 0; t < PARTS + 1; ++t) {
              const uint32_t qa = tmem + CHUNK_T_Q + (t == 0 ? HD / 2 : 0);
              const uint32_t bb = b0 + (PARTS == 2 && t == 1 ? PART : 0);
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) {
                mma_f16_ts(d, qa + k * 8, gemm::smem_desc(bb + k * 2 * BN * 16, BN * 16, 128),
                           IDESC_S, acc);
                acc = true;
              }
            }
            mma_commit(&sh->s_full[w]);
            mma_commit(&sh->empty[slot]);
            any = true;
            ++cnt[w];
            ++it;
          }
          if (j >= 1) {
            const int w = (j - 1) & 1, slot = it % NS;
            ok = wait(&sh->full[slot], it / NS, 45);
            if (ok) ok = wait(&sh->p_full[w], pcnt[w], 46);
            if (ok && pcnt[w] > 0) ok = wait(&sh->o_free[w], pcnt[w] - 1, 47);
            if (!ok) break;
            tc_fence_after();
            const uint32_t b0 = smem_u32(ring + (size_t)slot * SLOT);
            const uint32_t pw = tmem + CHUNK_T_S + w * BN;
            const uint32_t d = tmem + CHUNK_T_O + w * 128;
            bool acc = false;
#pragma unroll
            for (int t = 0; t < PARTS + 1; ++t) {
              const uint32_t bb = b0 + (PARTS == 2 && t == 1 ? PART : 0);
#pragma unroll
              for (int k = 0; k < BN / 16; ++k) {
                // weights of 32 keys: 16 columns hi, 16 lo
                const uint32_t pa = pw + (k / 2) * 32 + (t == 0 ? 16 : 0) + (k & 1) * 8;
                mma_f16_ts(d, pa, gemm::smem_desc(bb + k * 256, 128, BN * 16), IDESC_O, acc);
                acc = true;
              }
            }
            mma_commit(&sh->o_full[w]);
            mma_commit(&sh->empty[slot]);
            ++pcnt[w];
            ++it;
          }
        }
      }
      if (any) {  // every product issued has completed before the memory goes
        mma_commit(&sh->drain);
        int dummy = 0;
        mbar_wait(&sh->drain, 0, &dummy, a.res, 48, a.wait_ns);
      }
    }
    __syncwarp();
  }
  } else {
    // ---- softmax groups -----------------------------------------------------
    regs_inc<192>();
    const int w = warp >> 2;             // group
    const int row = threadIdx.x & 127;   // row = lane of tensor memory
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + CHUNK_T_S + w * BN, t_o = t_lane + CHUNK_T_O + w * 128;
    const uint32_t t_ox = t_lane + CHUNK_T_O + (w ^ 1) * 128;
    float* tb = tbuf + warp * 32 * 33;
    int done = 0;  // tiles of this group so far
    bool ok = true;
    if (threadIdx.x == 0) a.split[blockIdx.x * 8] = 0;
    for (; more && ok; more = chunk_next(a, sh, c)) {
      const int n = c.j1 - c.j0;
      const int ntok = min(tt, c.q.n_q - c.rt * tt);
      const int live_rows = ntok * a.group;
      const bool warp_live = (warp & 3) * 32 < live_rows;
      const bool live = row < live_rows;
      // keys this row sees in all
      const int see = live ? c.q.kv_len - c.q.n_q + c.rt * tt + row / a.group + 1 : 0;
      const long long row0 = (long long)c.q.q0 + c.rt * tt;
      const float* qrow = a.q + (row0 + row / a.group) * a.ldq +
                          (size_t)(c.kvh * a.group + row % a.group) * HD;
      float sc = 0.0f;
      if (warp_live) {
        // q rows: read by rows, turned in shared memory to one row per lane
        float qv[HD];
        float m = 0.0f;
#pragma unroll
        for (int dc = 0; dc < HD; dc += 32) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rl = i * 4 + (lane >> 3), r = (warp & 3) * 32 + rl;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < live_rows)
              x = *reinterpret_cast<const float4*>(
                  a.q + (row0 + r / a.group) * a.ldq +
                  (size_t)(c.kvh * a.group + r % a.group) * HD + dc + (lane & 7) * 4);
            float* t = tb + rl * 33 + (lane & 7) * 4;
            t[0] = x.x;
            t[1] = x.y;
            t[2] = x.z;
            t[3] = x.w;
          }
          __syncwarp();
#pragma unroll
          for (int d = 0; d < 32; ++d) {
            qv[dc + d] = tb[lane * 33 + d];
            m = fmaxf(m, fabsf(qv[dc + d]));
          }
        }
        const int e2 = exp_of(m);  // the row's largest value lands in [2^10, 2^11)
        const float up = pow2i(10 - e2);
        sc = a.scale * pow2i(e2 - 10 < -126 ? -126 : e2 - 10);
#pragma unroll
        for (int dc = 0; dc < HD; dc += 32) {
          uint32_t u[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = qv[dc + 2 * i] * up, y = qv[dc + 2 * i + 1] * up;
            u[i] = pack_h2(x, y);
            if (w == 1) {  // group 0 stores hi, group 1 lo
              const float2 b = unpack_h2(u[i]);
              u[i] = pack_h2(x - b.x, y - b.y);
            }
          }
          tmem_st16(t_lane + CHUNK_T_Q + w * (HD / 2) + dc / 2, u);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->q_ready);

      float o[HD], m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int d = 0; d < HD; ++d) o[d] = 0.0f;
      for (int j = w; j < n; j += 2, ++done) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->s_full[w], done & 1, &sh->abort_flag, a.res,
                                               49, a.wait_ns));
        if (!ok) break;
        tc_fence_after();
        const int kb = (c.j0 + j) * BN;
        const int seen = see - kb < 0 ? 0 : see - kb > BN ? BN : see - kb;
        float corr = 1.0f, vs = 1.0f;
        const bool whole = __all_sync(0xffffffffu, seen == BN || !live);
        // the tile's K and V among the loaded items (a loader is at most NS + 4
        // items ahead of the softmax groups)
        const int item0 = 2 * (int)(c.unit + c.j0 - sh->begin);
        const int item_k = item0 + (j == 0 ? 0 : 2 * j - 1);
        const int item_v = item0 + (j == n - 1 ? 2 * n - 1 : 2 * j + 2);
        if (warp_live) {
          float ks = sc;
          if constexpr (ES == 4) ks *= *(volatile float*)&sh->scale[item_k & 31];
          float mx = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[32];
            tmem_ld32(t_s + h * 32, v);
            tmem_wait_ld();
            if (whole) {
#pragma unroll
              for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(v[i]));
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (h * 32 + i < seen) mx = fmaxf(mx, __uint_as_float(v[i]));
            }
          }
          const float mn = fmaxf(m, mx * ks);
          const float mu = mn == -INFINITY ? 0.0f : mn;
          corr = m == -INFINITY ? 0.0f : ex2(m - mu);
          m = mn;
          const float off = 13.0f - mu;
          float sum = 0.0f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[32];
            tmem_ld32(t_s + h * 32, v);
            tmem_wait_ld();
            uint32_t ph[16], pl[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x = ex2(fmaf(__uint_as_float(v[2 * i]), ks, off));
              float y = ex2(fmaf(__uint_as_float(v[2 * i + 1]), ks, off));
              if (!whole) {
                if (h * 32 + 2 * i >= seen) x = 0.0f;
                if (h * 32 + 2 * i + 1 >= seen) y = 0.0f;
              }
              sum += x;
              sum += y;
              ph[i] = pack_h2(x, y);
              const float2 b = unpack_h2(ph[i]);
              pl[i] = pack_h2(x - b.x, y - b.y);
            }
            tmem_st16(t_s + h * 32, ph);
            tmem_st16(t_s + h * 32 + 16, pl);
          }
          l = fmaf(l, corr, sum);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[w]);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->o_full[w], done & 1, &sh->abort_flag, a.res,
                                               50, a.wait_ns));
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          if constexpr (ES == 4) vs = *(volatile float*)&sh->scale[item_v & 31];
#pragma unroll
          for (int dc = 0; dc < HD; dc += 32) {
            uint32_t v[32];
            tmem_ld32(t_o + dc, v);
            tmem_wait_ld();
            float scale_v = vs;
            if (!whole && live && seen < BN) {
              bool odd = false;
#pragma unroll
              for (int i = 0; i < 32; ++i) odd |= !(fabsf(__uint_as_float(v[i])) <= 3.4028235e38f);
              if (odd) {  // an unseen NaN or infinity
                const int page = seen > 0 ? c.q.pages[((size_t)a.layer * a.hkv + c.kvh) * c.q.pps +
                                                      kb / KV_PAGE]
                                          : 0;
                const bool in = page >= 0 && page < c.q.n_pages;
                const KT* rows = reinterpret_cast<const KT*>(c.q.pool) +
                                 ((size_t)(in ? page : 0) * KV_PAGE + (kb & (KV_PAGE - 1))) * 2 * HD;
                chunk_row_slow<HD, KT>(rows, in ? seen : 0, qrow, a.scale, m, dc, tb + lane * 33);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(tb[lane * 33 + i]);
                scale_v = 1.0f;
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[dc + i] = fmaf(__uint_as_float(v[i]), scale_v, o[dc + i] * corr);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->o_free[w]);
      }
      if (!ok) break;

      // the groups swap halves of their outputs through tensor memory: group 0
      // finishes dims [0, HD / 2), group 1 the others
      constexpr int HH = HD / 2;
      if (w >= n) {  // no tile of this segment waited for the others to leave the last one
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->q_ready, c.seg & 1, &sh->abort_flag, a.res, 52,
                                               a.wait_ns));
        if (!ok) break;
      }
      if (warp_live) {
        sh->ml[w][row][0] = m;
        sh->ml[w][row][1] = l;
#pragma unroll
        for (int dc = 0; dc < HH; dc += 16) {
          uint32_t u[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            u[i] = __float_as_uint(w == 0 ? o[HH + dc + i] : o[dc + i]);
          tmem_st16(t_o + dc, u);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->xchg);
      ok = __all_sync(0xffffffffu, mbar_wait(&sh->xchg, c.seg & 1, &sh->abort_flag, a.res, 51,
                                             a.wait_ns));
      if (!ok) break;
      tc_fence_after();
      const bool split = c.j0 > 0 || c.j1 < c.nk;
      const bool bad = *(volatile int*)&sh->bad[c.seg & 15] == c.seg + 1;
      // a piece that begins its row tile goes to the CTA's second place
      const size_t place = 2 * (size_t)blockIdx.x + (c.j0 == 0 ? 1 : 0);
      if (warp_live) {
        const float m2 = sh->ml[w ^ 1][row][0], l2 = sh->ml[w ^ 1][row][1];
        const float M = fmaxf(m, m2);
        const float f = m == -INFINITY ? 0.0f : ex2(m - M);
        const float f2 = m2 == -INFINITY ? 0.0f : ex2(m2 - M);
        const float L = fmaf(l, f, l2 * f2);
        const float inv = split ? 1.0f : L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
        if (split && live && w == 0) {
          a.part_ml[(place * CHUNK_BM + row) * 2] = bad ? __int_as_float(0x7fc00000) : M;
          a.part_ml[(place * CHUNK_BM + row) * 2 + 1] = L;
        }
        constexpr int OC = HH < 32 ? HH : 32;  // dims written at a time
#pragma unroll
        for (int dc = 0; dc < HH; dc += OC) {
#pragma unroll
          for (int e = 0; e < OC; e += 16) {
            uint32_t v[16];
            tmem_ld16(t_ox + dc + e, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float mine = w == 0 ? o[dc + e + i] : o[HH + dc + e + i];
              tb[lane * 33 + e + i] = fmaf(__uint_as_float(v[i]), f2, mine * f) * inv;
            }
          }
          __syncwarp();
          constexpr int LPR = OC / 4;  // lanes per row
#pragma unroll
          for (int i = 0; i < LPR; ++i) {
            const int rl = i * (32 / LPR) + lane / LPR, r = (warp & 3) * 32 + rl;
            const float* t = tb + rl * 33 + (lane % LPR) * 4;
            const float4 x = make_float4(t[0], t[1], t[2], t[3]);
            const int d = w * HH + dc + (lane % LPR) * 4;
            if (r < live_rows) {
              if (split)
                *reinterpret_cast<float4*>(a.part_o + (place * CHUNK_BM + r) * HD + d) = x;
              else if (!bad)
                *reinterpret_cast<float4*>(a.out + (row0 + r / a.group) * a.ldo +
                                           (size_t)(c.kvh * a.group + r % a.group) * HD + d) = x;
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      if (threadIdx.x == 0 && split && c.j1 == c.nk) {
        // this CTA ends the row tile: what k_chunk_merge joins
        const long long sum = sh->pre[a.n_seqs];
        long long ctas = (sum + CHUNK_MIN_TILES - 1) / CHUNK_MIN_TILES;
        if (ctas > (long long)gridDim.x) ctas = gridDim.x;
        int* d = a.split + blockIdx.x * 8;
        d[0] = live_rows;
        d[1] = chunk_owner(c.unit, sum, (int)ctas);
        d[2] = c.s;
        d[3] = c.kvh;
        d[4] = c.rt;
      }
    }
  }
  cp_async_wait<0>();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 15) {
    __syncwarp();
    tmem_dealloc(tmem, CHUNK_T_COLS);
  }
}

// Joins the pieces of a row tile that several CTAs hold, in the order of the
// CTAs: out = sum O_p 2^(m_p - M) / sum l_p 2^(m_p - M).  grid (CTAs of the
// attention, row slices), 256 threads; a block takes its rows one by one, its
// warps the row's pieces.
template <int HD>
__global__ void __launch_bounds__(256) k_chunk_merge(const __grid_constant__ ChunkArgs a) {
  __shared__ float sm_o[8][HD], sm_l[8], sm_m[8];
  const int* d = a.split + blockIdx.x * 8;
  const int live = d[0];
  if (live == 0) return;
  const int c0 = d[1], c1 = blockIdx.x, n = c1 - c0 + 1;
  const l3g_chunk_seq q = a.seqs[d[2]];
  const int kvh = d[3], tt = CHUNK_BM / a.group;
  const long long row0 = (long long)q.q0 + (long long)d[4] * tt;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int V = HD / 32;
  for (int r = blockIdx.y; r < live; r += gridDim.y) {
    float M = -INFINITY, L = 0.0f, o[V];
    bool bad = false;  // a maximum that is NaN marks a piece with a page outside its pool
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.0f;
    for (int p = warp; p < n; p += 8) {
      const size_t place = 2 * (size_t)(c0 + p) + (p == 0 ? 1 : 0);
      const float m = a.part_ml[(place * CHUNK_BM + r) * 2];
      const float l = a.part_ml[(place * CHUNK_BM + r) * 2 + 1];
      bad |= m != m;
      const float mn = fmaxf(M, m);
      const float f = M == -INFINITY ? 0.0f : ex2(M - mn);
      const float g = m == -INFINITY ? 0.0f : ex2(m - mn);
      M = mn;
      L = fmaf(L, f, l * g);
#pragma unroll
      for (int i = 0; i < V; ++i)
        o[i] = fmaf(o[i], f, a.part_o[(place * CHUNK_BM + r) * HD + i * 32 + lane] * g);
    }
    if (lane == 0) {
      sm_m[warp] = bad ? __int_as_float(0x7fc00000) : M;
      sm_l[warp] = L;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sm_o[warp][i * 32 + lane] = o[i];
    __syncthreads();
    if (threadIdx.x < HD) {
      M = -INFINITY;
      bad = false;
      for (int w = 0; w < 8; ++w) {
        bad |= sm_m[w] != sm_m[w];
        M = fmaxf(M, sm_m[w]);
      }
      float O = 0.0f;
      L = 0.0f;
      for (int w = 0; w < 8; ++w) {
        const float f = sm_m[w] == -INFINITY ? 0.0f : ex2(sm_m[w] - M);
        L = fmaf(sm_l[w], f, L);
        O = fmaf(sm_o[w][threadIdx.x], f, O);
      }
      if (!bad)
        a.out[(row0 + r / a.group) * a.ldo + (size_t)(kvh * a.group + r % a.group) * HD +
              threadIdx.x] = L > 0.0f ? O / L : L == 0.0f ? 0.0f : L;
    }
    __syncthreads();
  }
}
