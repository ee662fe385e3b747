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
// keys per tile (divides KV_PAGE): 128 of an f16 cache; 64 of an f32 cache,
// whose tiles take twice the shared memory
__host__ __device__ constexpr int chunk_bn(int es) { return es == 2 ? 128 : 64; }
constexpr int CHUNK_SOFT = 8;       // softmax warps: two groups of four
constexpr int CHUNK_LOAD = 7;       // loader warps
constexpr int CHUNK_THREADS = 32 * (CHUNK_SOFT + CHUNK_LOAD + 1);
constexpr int CHUNK_MIN_KEYS = 256;  // keys a CTA takes at least
__host__ __device__ constexpr int chunk_min_tiles(int bn) { return CHUNK_MIN_KEYS / bn; }
// tensor-memory columns: scores / weights of the two groups (at most 128
// each), q hi and lo (64 each), the tile output
constexpr uint32_t CHUNK_T_S = 0, CHUNK_T_Q = 256, CHUNK_T_O = 384, CHUNK_T_COLS = 512;

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
  uint8_t* maps;     // [grid][CHUNK_LOAD][128] the loaders' tensor maps
  Result* res;
  unsigned long long wait_ns;
  // a pool as rows of 2 HD elements, boxes of one panel of a key tile; its base
  // address is replaced by each sequence's pool
  CUtensorMap map;
};

// (see chunk_open)
struct ChunkCursor {
  long long pos, unit;  // next tile, first tile of its row tile
  int s, kvh, rt, seg;
  l3g_chunk_seq q;      // the sequence's descriptor
  int nk, j0, j1;
};

struct ChunkSmem {
  uint8_t map[CHUNK_LOAD][128];  // (at the start: 128-byte aligned)
  uint64_t full[CHUNK_LOAD], empty[CHUNK_LOAD], raw[CHUNK_LOAD];  // K / V slots
  uint64_t s_full[2], p_full[2], o_full[2], o_free[2];
  uint64_t q_ready, xchg, drain;
  uint32_t tmem_base;
  int abort_flag;
  int n_tiles_lo, pad;
  long long begin, end;          // the CTA's range of the linear tile order
  long long unit0;               // first tile of the unit that holds `begin`
  int s0, kvh0, rt0, per;
  int bad[16];                   // segment + 1 whose pages are out of bounds
  float scale[32];               // f32 caches: 2^e of the items' tiles, item & 31
  ChunkCursor cur[CHUNK_SOFT];   // the softmax warps' cursors, out of their registers
  float ml[2][CHUNK_BM][2];      // the groups' statistics
  long long pre[L3G_CHUNK_SEQS_MAX + 1];  // tiles before each sequence
};
constexpr int CHUNK_HEAD = 14 * 1024;
static_assert(sizeof(ChunkSmem) <= CHUNK_HEAD, "chunk attention smem head");
constexpr int CHUNK_TBUF = 32 * 33 * 4;  // a softmax warp's transposition buffer
__host__ __device__ constexpr int chunk_slot_bytes(int hd, int es) {
  return chunk_bn(es) * hd * es;  // f16: one operand tile; f32: its hi and lo tiles
}
// one slot per loader warp, as far as they fit
__host__ __device__ constexpr int chunk_slots(int hd, int es) {
  return (180 * 1024) / chunk_slot_bytes(hd, es) < CHUNK_LOAD
             ? (180 * 1024) / chunk_slot_bytes(hd, es)
             : CHUNK_LOAD;
}
__host__ __device__ constexpr int chunk_ring_off() {
  return (CHUNK_HEAD + CHUNK_SOFT * CHUNK_TBUF + 1023) / 1024 * 1024;
}
// Operand tiles in shared memory: panels of up to 64 dims, [key][row bytes] with
// the 16-byte pieces of a row swizzled by the key (the tensor core's 128-byte
// and 64-byte swizzles), keys in groups of 8 one after another.  An f32 cache's
// panel is fetched as two raw panels of 32 floats, and each key's two raw rows
// become its hi and lo rows in place; with 32 dims a row holds hi, then lo.
__host__ __device__ constexpr int chunk_row_bytes(int hd, int es) {
  return es == 2 && hd < 64 ? 64 : 128;
}
__host__ __device__ constexpr int chunk_box_cols(int hd, int es) {  // elements of a box's row
  return es == 4 ? 32 : hd < 64 ? 32 : 64;
}
// byte of 16-byte piece `piece` of key k in a panel of rows of rb bytes
__host__ __device__ constexpr int chunk_piece(int rb, int k, int piece) {
  return k * rb + ((piece ^ (rb == 128 ? k & 7 : (k >> 1) & 3)) << 4);
}
__host__ __device__ constexpr int chunk_smem_bytes(int hd, int es) {
  return chunk_ring_off() + chunk_slots(hd, es) * chunk_slot_bytes(hd, es);
}

// Bounded wait as mbar_wait, for waits that are on the critical path many
// times: the thread is suspended by the hardware (polling warps would take
// issue slots from the others), 20 us a try, and the timer, which takes longer
// to read than most of the waits, is looked at every 16th try.
__device__ __forceinline__ bool chunk_wait(uint64_t* b, uint32_t parity, ChunkSmem* sh,
                                           const ChunkArgs& a, int where) {
  uint64_t t0 = 0;
  for (int i = 0; !mbar_try_wait(b, parity, 20000); ++i) {
    if (*(volatile int*)&sh->abort_flag) return false;
    if ((i & 15) == 15) {
      const uint64_t t = gtime();
      if (t0 == 0) t0 = t;
      if (t - t0 > a.wait_ns) {
        *(volatile int*)&sh->abort_flag = 1;
        report(a.res, ERR_TIMEOUT, where);
        return false;
      }
    }
  }
  return true;
}

// Whether a descriptor stays inside its bounds (its pages are checked where
// they are read).
__device__ __forceinline__ bool chunk_seq_ok(const l3g_chunk_seq& s, int total_q) {
  return s.pool && s.pages && s.pps >= 0 && s.q0 >= 0 && s.n_q >= 0 && s.n_q <= total_q &&
         s.q0 <= total_q - s.n_q && s.kv_len >= 0 &&
         (long long)s.kv_len <= (long long)s.pps * KV_PAGE;
}
// Key tiles of row tile rt (at least one: a row that sees nothing is written)
template <int BN>
__device__ __forceinline__ int chunk_tiles(const l3g_chunk_seq& s, int tt, int rt) {
  const long long end = (long long)(rt + 1) * tt;
  const long long see = (long long)s.kv_len - s.n_q + (end < s.n_q ? end : s.n_q);
  return see <= BN ? 1 : (int)((see + BN - 1) / BN);
}

// The CTAs share the linear order (sequence, kv head, row tile, key tile) in
// equal ranges; a row tile whose keys several CTAs hold is joined by
// k_chunk_merge.  A cursor walks a CTA's range in segments, each the key tiles
// [j0, j1) of one row tile.
template <int BN>
__device__ __forceinline__ void chunk_open(const ChunkArgs& a, ChunkCursor& c, long long end) {
  c.nk = chunk_tiles<BN>(c.q, CHUNK_BM / a.group, c.rt);
  c.j0 = (int)(c.pos - c.unit);
  c.j1 = (int)(end - c.unit < c.nk ? end - c.unit : c.nk);
}
template <int BN>
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
  chunk_open<BN>(a, c, sh->end);
  return true;
}
template <int BN>
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
  chunk_open<BN>(a, c, sh->end);
  return true;
}

// Warp 0: the tiles of every sequence, then this CTA's range and where it starts.
template <int BN>
__device__ __forceinline__ void chunk_plan(const ChunkArgs& a, ChunkSmem* sh, int lane) {
  const int tt = CHUNK_BM / a.group;
  long long sum = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    const int s = s0 + lane;
    long long n = 0;
    if (s < a.n_seqs) {
      const l3g_chunk_seq q = a.seqs[s];
      if (chunk_seq_ok(q, a.total_q)) {
        for (int rt = 0; rt < (q.n_q + tt - 1) / tt; ++rt) n += chunk_tiles<BN>(q, tt, rt);
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
    long long ctas = (sum + chunk_min_tiles(BN) - 1) / chunk_min_tiles(BN);
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
        const int nk = chunk_tiles<BN>(q, tt, rt);
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

// o[d] = sum_j p_j V_j[d0 + d], d < 16, over the n keys of `rows` that a row
// sees, in fp32 from the cache itself: for a tile whose unseen keys hold a NaN
// or an infinity, which the product would multiply by zero.  o is shared
// memory of this thread's own; small loops, as it hardly ever runs.
template <int HD, typename KT>
__device__ __forceinline__ void chunk_row_slow(const KT* rows, int n, const float* q, float scale,
                                               float m, int d0, float* o) {
#pragma unroll 1
  for (int d = 0; d < 16; ++d) o[d] = 0.0f;
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const KT* k = rows + (size_t)j * 2 * HD;
    float s = 0.0f;
#pragma unroll 1
    for (int d = 0; d < HD; ++d) s = fmaf(q[d], (float)k[d], s);
    const float p = ex2(fmaf(s, scale, 13.0f - m));
#pragma unroll 1
    for (int d = 0; d < 16; ++d) o[d] = fmaf(p, (float)k[HD + d0 + d], o[d]);
  }
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
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
// Either tile is panels of [key][dims], swizzled (chunk_piece).
template <int HD, typename KT>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
    k_chunk_attention(const __grid_constant__ ChunkArgs a) {
  constexpr int ES = (int)sizeof(KT);
  constexpr int BN = chunk_bn(ES);
  constexpr int NS = chunk_slots(HD, ES);
  constexpr int SLOT = chunk_slot_bytes(HD, ES);
  constexpr int PARTS = ES == 4 ? 2 : 1;       // terms per operand: hi (, lo)
  constexpr int RB = chunk_row_bytes(HD, ES);  // row bytes of a panel
  constexpr int BOX = BN * RB;                 // bytes of a panel
  constexpr int PANELS = SLOT / BOX;           // boxes per tile
  // bytes from an operand's hi to its lo, and from 64 dims to the next 64
  constexpr int LO = ES == 4 ? (HD == 32 ? 64 : BOX) : 0;
  constexpr int NEXT = PARTS * BOX;
  L3G_DYNAMIC_SMEM(smem);
  ChunkSmem* sh = reinterpret_cast<ChunkSmem*>(smem);
  float* tbuf = reinterpret_cast<float*>(smem + CHUNK_HEAD);
  uint8_t* ring = smem + chunk_ring_off();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tt = CHUNK_BM / a.group;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->empty[i], 1);
      mbar_init(&sh->raw[i], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh->s_full[w], 1);
      mbar_init(&sh->p_full[w], 4);
      mbar_init(&sh->o_full[w], 1);
      mbar_init(&sh->o_free[w], 4);
    }
    mbar_init(&sh->q_ready, CHUNK_SOFT);
    mbar_init(&sh->xchg, CHUNK_SOFT);
    mbar_init(&sh->drain, 1);
    sh->abort_flag = 0;
    for (int i = 0; i < 16; ++i) sh->bad[i] = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    __syncwarp();
    chunk_plan<BN>(a, sh, lane);
  }
  if (warp == 15) tmem_alloc(&sh->tmem_base, CHUNK_T_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;

  // two warpgroups give 64 of their 128 registers a thread to the other two
  if (warp >= CHUNK_SOFT) {
  regs_dec<64>();
  if (warp < CHUNK_SOFT + CHUNK_LOAD) {
    // ---- loaders ----------------------------------------------------------
    // Warp lw brings the items lw, lw + NS, ... whole into slot lw: a tile whose
    // keys all exist by tensor copies (one box per panel), the last, part-filled
    // one by 16-byte copies with zeros for the keys past the cache's end.
    const int lw = warp - CHUNK_SOFT;
    const int kl = lane >> 3, cl = lane & 7;  // key and piece of the lane
    uint8_t* map = a.maps + ((size_t)blockIdx.x * CHUNK_LOAD + lw) * 128;
    const void* map_pool = nullptr;
    uint8_t* const dst = ring + (size_t)lw * SLOT;
    int it = lw;                  // this warp's next item
    int it0 = 0;                  // the segment's first
    bool ok = lw < NS;
    ChunkCursor c;
    bool more = chunk_first<BN>(a, sh, c);
    for (; more && ok; more = chunk_next<BN>(a, sh, c)) {
      const int n = c.j1 - c.j0;
      const int* pages = c.q.pages + ((size_t)a.layer * a.hkv + c.kvh) * c.q.pps;
      for (; it < it0 + 2 * n; it += NS) {
        const int i = it - it0;
        const bool is_v = i == 2 * n - 1 || (i > 0 && i % 2 == 0);
        const int j = c.j0 + (i == 2 * n - 1 ? n - 1 : is_v ? i / 2 - 1 : (i + 1) / 2);
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
        const int use = it / NS;
        if (use > 0) {
          ok = __all_sync(0xffffffffu, chunk_wait(&sh->empty[lw], (use - 1) & 1, sh, a, 40));
          if (!ok) break;
        }
        // (after the wait: the slot's last copy, which used the map, is over)
        if (cnt == BN && map_pool != c.q.pool) {
          map_pool = c.q.pool;
          tmap_rebase(map, sh->map[lw], &a.map, map_pool, lane);
        }
        uint64_t* landed = ES == 2 ? &sh->full[lw] : &sh->raw[lw];
        if (cnt == BN) {
          if (lane == 0) {
            mbar_arrive_expect_tx(landed, SLOT);
            const int x = is_v ? HD : 0, y = page * KV_PAGE + (kb & (KV_PAGE - 1));
#pragma unroll
            for (int p = 0; p < PANELS; ++p)
              tma_load_2d(dst + p * BOX, map, x + p * chunk_box_cols(HD, ES), y, landed);
          }
        } else {
          const uint8_t* src =
              reinterpret_cast<const uint8_t*>(c.q.pool) +
              (((size_t)page * KV_PAGE + (kb & (KV_PAGE - 1))) * 2 + (is_v ? 1 : 0)) * HD * ES;
          constexpr int PIECES = RB / 16;  // per row
#pragma unroll 1
          for (int e = lane; e < PANELS * BN * PIECES; e += 32) {
            const int p = e / (BN * PIECES), k = e / PIECES % BN, pc = e % PIECES;
            const bool in = k < cnt;
            cp_async16(dst + p * BOX + chunk_piece(RB, k, pc),
                       in ? src + (size_t)k * 2 * HD * ES + p * RB + pc * 16
                          : reinterpret_cast<const uint8_t*>(c.q.pool),
                       in ? 16u : 0u);
          }
          cp_async_commit();
          cp_async_wait<0>();
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(landed);
        }
        if constexpr (ES == 4) {
          ok = __all_sync(0xffffffffu, chunk_wait(&sh->raw[lw], use & 1, sh, a, 41));
          if (!ok) break;
          // the tile's scale, from its largest finite magnitude
          float m = 0.0f;
#pragma unroll 8
          for (int e = lane; e < SLOT / 16; e += 32) {
            const float4 x = reinterpret_cast<const float4*>(dst)[e];
            const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) {
              const float v = fabsf(f[i2]);
              m = v <= 3.4028235e38f ? fmaxf(m, v) : m;
            }
          }
          const int e2 = exp_of(warp_max(m));  // it lands in [2^14, 2^15)
          const float up = pow2i(14 - e2);
          if (lane == 0) sh->scale[it & 31] = 1.0f / up;
          __syncwarp();
          // 8 lanes take a key's raw row (32 dims) or rows (64), 4 dims of
          // each a lane, and put the two terms in their place
          constexpr int RAW = HD == 32 ? 1 : 2;  // raw rows that become hi and lo rows
#pragma unroll 1
          for (int p = 0; p < PANELS; p += RAW)
#pragma unroll 4
            for (int k0 = 0; k0 < BN; k0 += 4) {
              const int k = k0 + kl;
              uint8_t* row = dst + p * BOX;
              float4 x[RAW];
#pragma unroll
              for (int r = 0; r < RAW; ++r)
                x[r] = *reinterpret_cast<const float4*>(row + r * BOX + chunk_piece(128, k, cl));
              __syncwarp();
#pragma unroll
              for (int r = 0; r < RAW; ++r) {
                uint2 hi, lo;
                const float f0 = x[r].x * up, f1 = x[r].y * up, f2 = x[r].z * up, f3 = x[r].w * up;
                hi.x = pack_h2(f0, f1);
                hi.y = pack_h2(f2, f3);
                const float2 b0 = unpack_h2(hi.x), b1 = unpack_h2(hi.y);
                lo.x = pack_h2(f0 - b0.x, f1 - b0.y);
                lo.y = pack_h2(f2 - b1.x, f3 - b1.y);
                // dims 32 r + 4 cl .. of the 64 (or 32): 8 bytes of a 64-byte half row
                const int at = r * 64 + cl * 8;
                *reinterpret_cast<uint2*>(row + chunk_piece(128, k, at >> 4) + (at & 8)) = hi;
                if constexpr (RAW == 2)
                  *reinterpret_cast<uint2*>(row + BOX + chunk_piece(128, k, at >> 4) + (at & 8)) = lo;
                else
                  *reinterpret_cast<uint2*>(row + chunk_piece(128, k, (64 + at) >> 4) + (at & 8)) = lo;
              }
            }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->full[lw]);
        }
      }
      it0 += 2 * n;
    }
  } else {
    // ---- product issuer -----------------------------------------------------
    // f16 operands, f32 accumulators (bits 4-5 = 1), M >> 4 at 24, N >> 3 at
    // 17; B of the second product MN-major (bit 16)
    constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | (8u << 24);
    constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
    // descriptors: byte offsets >> 4; K steps within a tile add to the low word
    // (swizzle mode at bits 61-63: 2 for 128-byte rows, 4 for 64-byte rows);
    // 8 keys are 8 rows, 64 dims of N (V) a panel
    constexpr uint64_t SWZ = RB == 128 ? 2ull << 61 : 4ull << 61;
    constexpr uint64_t DESC_K = gemm::smem_desc(0, 16, 8 * RB) | SWZ;
    constexpr uint64_t DESC_V = gemm::smem_desc(0, NEXT, 8 * RB) | SWZ;
    const uint32_t ring0 = smem_u32(ring) >> 4;
    int it = 0;
    // tiles of group 0 and 1 so far, issued to S and to O, over all segments
    int s0 = 0, s1 = 0, o0 = 0, o1 = 0, last = -1;
    ChunkCursor c;
    bool more = chunk_first<BN>(a, sh, c);
    bool ok = true, any = false;
    // the whole warp walks the loop, one lane issues
    auto wait = [&](uint64_t* b, int phase, int site) {
      return __all_sync(0xffffffffu, chunk_wait(b, phase & 1, sh, a, site)) != 0;
    };
    for (; more && ok; more = chunk_next<BN>(a, sh, c)) {
      const int n = __shfl_sync(0xffffffffu, c.j1 - c.j0, 0);
      ok = wait(&sh->q_ready, c.seg, 42);
      if (!ok) break;
      tc_fence_after();
      for (int j = 0; j <= n && ok; ++j) {
        if (j < n) {
          const int w = j & 1, slot = it % NS;
          ok = wait(&sh->full[slot], it / NS, 43);
          // the weights of the group's previous tile lie over S until its
          // second product is complete
          const int before = w ? s1 : s0;
          if (ok && before > 0) ok = wait(&sh->o_full[w], before - 1, 44);
          if (!ok) break;
          tc_fence_after();
          const uint32_t b0 = ring0 + (uint32_t)(slot * (SLOT >> 4)) + (uint32_t)DESC_K;
          const uint32_t d = tmem + CHUNK_T_S + w * BN;
          if (elect_one()) {
            // small terms first: q_lo K_hi, (q_hi K_lo,) q_hi K_hi
#pragma unroll
            for (int t = 0; t < PARTS + 1; ++t) {
              const uint32_t qa = tmem + CHUNK_T_Q + (t == 0 ? HD / 2 : 0);
              const uint32_t bb = b0 + (PARTS == 2 && t == 1 ? LO >> 4 : 0);
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) {
                const uint32_t bk = bb + (k / 4) * (NEXT >> 4) + (k % 4) * 2;  // 16 dims: 32 bytes
                if (t == 0 && k == 0)
                  mma_f16_ts<false>(d, qa, bk, (uint32_t)(DESC_K >> 32), IDESC_S);
                else
                  mma_f16_ts<true>(d, qa + k * 8, bk, (uint32_t)(DESC_K >> 32), IDESC_S);
              }
            }
            mma_commit(&sh->s_full[w]);
            mma_commit(&sh->empty[slot]);
          }
          __syncwarp();
          any = true;
          if (w)
            ++s1;
          else
            ++s0;
          ++it;
        }
        if (j >= 1) {
          const int w = (j - 1) & 1, slot = it % NS;
          ok = wait(&sh->full[slot], it / NS, 45);
          if (ok) ok = wait(&sh->p_full[w], w ? o1 : o0, 46);
          // the output of the tile before, of group `last`, has been read
          if (ok && last >= 0) ok = wait(&sh->o_free[last], (last ? o1 : o0) - 1, 47);
          if (!ok) break;
          tc_fence_after();
          const uint32_t b0 = ring0 + (uint32_t)(slot * (SLOT >> 4)) + (uint32_t)DESC_V;
          const uint32_t pw = tmem + CHUNK_T_S + w * BN;
          const uint32_t d = tmem + CHUNK_T_O;
          if (elect_one()) {
#pragma unroll
            for (int t = 0; t < PARTS + 1; ++t) {
              const uint32_t bb = b0 + (PARTS == 2 && t == 1 ? LO >> 4 : 0);
#pragma unroll
              for (int k = 0; k < BN / 16; ++k) {
                // weights of 16 keys: 8 columns hi, 8 lo
                const uint32_t pa = pw + k * 16 + (t == 0 ? 8 : 0);
                if (t == 0 && k == 0)
                  mma_f16_ts<false>(d, pa, bb, (uint32_t)(DESC_V >> 32), IDESC_O);
                else
                  mma_f16_ts<true>(d, pa, bb + k * RB, (uint32_t)(DESC_V >> 32), IDESC_O);  // 16 keys
              }
            }
            mma_commit(&sh->o_full[w]);
            mma_commit(&sh->empty[slot]);
          }
          __syncwarp();
          if (w)
            ++o1;
          else
            ++o0;
          last = w;
          ++it;
        }
      }
    }
    if (any) {  // every product issued has completed before the memory goes
      if (elect_one()) mma_commit(&sh->drain);
      int dummy = 0;
      mbar_wait(&sh->drain, 0, &dummy, a.res, 48, a.wait_ns);
    }
    __syncwarp();
  }
  } else {
    // ---- softmax groups -----------------------------------------------------
    regs_inc<192>();
    const int w = warp >> 2;             // group
    const int row = threadIdx.x & 127;   // row = lane of tensor memory
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + CHUNK_T_S + w * BN, t_o = t_lane + CHUNK_T_O;
    const uint32_t t_mine = t_o + w * (HD / 2), t_theirs = t_o + (w ^ 1) * (HD / 2);
    float* tb = tbuf + warp * 32 * 33;
    int done = 0;    // tiles of this group so far
    int theirs = 0;  // ... of the other group
    bool ok = true;
    if (threadIdx.x == 0) a.split[blockIdx.x * 8] = 0;
    ChunkCursor& c = sh->cur[warp];
    bool more = false;
    if (lane == 0) more = chunk_first<BN>(a, sh, c);
    for (;;) {
      if (!__shfl_sync(0xffffffffu, more, 0)) break;
      __syncwarp();
      const int n = c.j1 - c.j0;
      const int ntok = min(tt, c.q.n_q - c.rt * tt);
      const int live_rows = ntok * a.group;
      const bool warp_live = (warp & 3) * 32 < live_rows;
      const bool live = row < live_rows;
      const int seg = c.seg;
      // keys this row sees in all
      const int see = live ? c.q.kv_len - c.q.n_q + c.rt * tt + row / a.group + 1 : 0;
      float sc = 0.0f;
      if (warp_live) {
        const long long row0 = (long long)c.q.q0 + c.rt * tt;
        // eight lanes read a row, four rows at a time, all in flight at once;
        // their hi (group 0) or lo (group 1) terms are turned in shared memory,
        // 64 dims at a time, to one row per lane
        const int rl4 = lane >> 3, l8 = lane & 7;
        float4 x[8][HD / 32];
        float up[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = (warp & 3) * 32 + i * 4 + rl4;
          const float* g = a.q + (row0 + r / a.group) * a.ldq +
                           (size_t)(c.kvh * a.group + r % a.group) * HD + l8 * 4;
#pragma unroll
          for (int k = 0; k < HD / 32; ++k)
            x[i][k] = r < live_rows ? *reinterpret_cast<const float4*>(g + k * 32)
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float m4 = 0.0f;
#pragma unroll
          for (int k = 0; k < HD / 32; ++k)
            m4 = fmaxf(fmaxf(fmaxf(m4, fabsf(x[i][k].x)), fmaxf(fabsf(x[i][k].y), fabsf(x[i][k].z))),
                       fabsf(x[i][k].w));
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m4 = fmaxf(m4, __shfl_xor_sync(0xffffffffu, m4, o));
          // the row's largest value lands in [2^10, 2^11); row i * 4 + k of the
          // warp is lane i * 4 + k's
          up[i] = pow2i(10 - exp_of(m4));
          const float mine = __shfl_sync(0xffffffffu, up[i], (lane & 3) * 8);
          if ((lane >> 2) == i) sc = a.scale / mine;
        }
        uint32_t* tw = reinterpret_cast<uint32_t*>(tb);
        constexpr int QH = HD < 64 ? HD : 64;  // dims at a time
#pragma unroll
        for (int h = 0; h < HD; h += QH) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < QH / 32; ++k) {
              const float4 y = x[i][h / 32 + k];
              uint32_t p0 = pack_h2(y.x * up[i], y.y * up[i]);
              uint32_t p1 = pack_h2(y.z * up[i], y.w * up[i]);
              if (w == 1) {
                const float2 b0 = unpack_h2(p0), b1 = unpack_h2(p1);
                p0 = pack_h2(fmaf(y.x, up[i], -b0.x), fmaf(y.y, up[i], -b0.y));
                p1 = pack_h2(fmaf(y.z, up[i], -b1.x), fmaf(y.w, up[i], -b1.y));
              }
              tw[(i * 4 + rl4) * 33 + k * 16 + l8 * 2] = p0;
              tw[(i * 4 + rl4) * 33 + k * 16 + l8 * 2 + 1] = p1;
            }
          __syncwarp();
#pragma unroll
          for (int e = 0; e < QH / 2; e += 16) {
            uint32_t u[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) u[i] = tw[lane * 33 + e + i];
            tmem_st16(t_lane + CHUNK_T_Q + w * (HD / 2) + h / 2 + e, u);
          }
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->q_ready);

      unsigned long long o2[HD / 2];  // the output, dims 2 i and 2 i + 1
      float m = -INFINITY, l = 0.0f;
      const int seen0 = see - c.j0 * BN;  // keys from the segment's first on that the row sees
#pragma unroll
      for (int d = 0; d < HD / 2; ++d) o2[d] = 0ull;
      for (int j = w; j < n; j += 2, ++done) {
        ok = __all_sync(0xffffffffu, chunk_wait(&sh->s_full[w], done & 1, sh, a, 49));
        if (!ok) break;
        tc_fence_after();
        const int seen = min(max(seen0 - j * BN, 0), BN);
        float corr = 1.0f, vs = 1.0f;
        const bool whole = __all_sync(0xffffffffu, seen == BN || !live);
        // the tile's K and V among the loaded items (a loader is at most NS + 4
        // items ahead of the softmax groups)
        const int item0 = ES == 4 ? 2 * (int)(c.unit + c.j0 - sh->begin) : 0;
        const int item_k = item0 + (j == 0 ? 0 : 2 * j - 1);
        const int item_v = item0 + (j == n - 1 ? 2 * n - 1 : 2 * j + 2);
        if (warp_live) {
          float ks = sc;
          if constexpr (ES == 4) ks *= *(volatile float*)&sh->scale[item_k & 31];
          // both passes over the scores load 16 columns ahead
          float mx = -INFINITY;
          uint32_t v0[16], v1[16];
          tmem_ld16(t_s, v0);
          tmem_wait_ld16(v0);
          if (whole) {
            float m2 = -INFINITY;
#pragma unroll 1
            for (int h = 0; h < BN; h += 32) {
              tmem_ld16(t_s + h + 16, v1);
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                mx = max3(mx, __uint_as_float(v0[i]), __uint_as_float(v0[i + 1]));
                m2 = max3(m2, __uint_as_float(v0[i + 2]), __uint_as_float(v0[i + 3]));
              }
              tmem_wait_ld16(v1);
              tmem_ld16(t_s + ((h + 32) & (BN - 1)), v0);  // at the end: the first again
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                mx = max3(mx, __uint_as_float(v1[i]), __uint_as_float(v1[i + 1]));
                m2 = max3(m2, __uint_as_float(v1[i + 2]), __uint_as_float(v1[i + 3]));
              }
              tmem_wait_ld16(v0);
            }
            mx = fmaxf(mx, m2);
          } else {
#pragma unroll 1
            for (int h = 0; h < BN; h += 16) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (h + i < seen) mx = fmaxf(mx, __uint_as_float(v0[i]));
              tmem_ld16(t_s + ((h + 16) & (BN - 1)), v0);
              tmem_wait_ld16(v0);
            }
          }
          const float mn = fmaxf(m, mx * ks);
          const float mu = mn == -INFINITY ? 0.0f : mn;
          corr = m == -INFINITY ? 0.0f : ex2(m - mu);
          m = mn;
          const float off = 13.0f - mu;
          const unsigned long long ks2 = pk2(ks, ks), off2 = pk2(off, off);
          const unsigned long long neg2 = pk2(-1.0f, -1.0f);
          unsigned long long sum = 0ull, sum2 = 0ull;  // pairs of fp32
          // weights of 16 keys from their scores v, stored over them
          auto weigh = [&](const uint32_t* v, int h) {
            uint32_t ph[8], pl[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 t = upk2(
                  fma2(pk2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ks2, off2));
              float x = ex2(t.x), y = ex2(t.y);
              if (!whole) {
                if (h + 2 * i >= seen) x = 0.0f;
                if (h + 2 * i + 1 >= seen) y = 0.0f;
              }
              const unsigned long long p2 = pk2(x, y);
              if (i & 1)
                sum2 = add2(sum2, p2);
              else
                sum = add2(sum, p2);
              ph[i] = pack_h2(x, y);
              const float2 b = unpack_h2(ph[i]);
              const float2 r = upk2(fma2(pk2(b.x, b.y), neg2, p2));
              pl[i] = pack_h2(r.x, r.y);
            }
            tmem_st8(t_s + h, ph);
            tmem_st8(t_s + h + 8, pl);
          };
#pragma unroll 1
          for (int h = 0; h < BN; h += 32) {
            tmem_ld16(t_s + h + 16, v1);
            weigh(v0, h);
            tmem_wait_ld16(v1);
            if (h + 32 < BN) tmem_ld16(t_s + h + 32, v0);
            weigh(v1, h + 16);
            tmem_wait_ld16(v0);
          }
          const float2 total = upk2(add2(sum, sum2));
          l = fmaf(l, corr, total.x + total.y);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[w]);
        ok = __all_sync(0xffffffffu, chunk_wait(&sh->o_full[w], done & 1, sh, a, 50));
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          if constexpr (ES == 4) vs = *(volatile float*)&sh->scale[item_v & 31];
          bool odd = false;
          if (!whole) {  // did an unseen NaN or infinity come in?
#pragma unroll 1
            for (int dc = 0; dc < HD; dc += 16) {
              uint32_t v[16];
              tmem_ld16(t_o + dc, v);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                odd |= !(fabsf(__uint_as_float(v[i])) <= 3.4028235e38f);
            }
            odd = odd && live && seen < BN;
          }
          if (__any_sync(0xffffffffu, odd)) {
            const int kb = (c.j0 + j) * BN;
            const float* qrow = a.q + ((long long)c.q.q0 + c.rt * tt + row / a.group) * a.ldq +
                                (size_t)(c.kvh * a.group + row % a.group) * HD;
            int page = 0;
            if (seen > 0)
              page = c.q.pages[((size_t)a.layer * a.hkv + c.kvh) * c.q.pps + kb / KV_PAGE];
            const bool in = page >= 0 && page < c.q.n_pages;
            const KT* rows = reinterpret_cast<const KT*>(c.q.pool) +
                             ((size_t)(in ? page : 0) * KV_PAGE + (kb & (KV_PAGE - 1))) * 2 * HD;
#pragma unroll 1
            for (int dc = 0; dc < HD; dc += 16) {
              uint32_t v[16];
              tmem_ld16(t_o + dc, v);
              tmem_wait_ld();
              if (odd) {
                chunk_row_slow<HD, KT>(rows, in ? seen : 0, qrow, a.scale, m, dc, tb + lane * 33);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(tb[lane * 33 + i] / vs);
              }
              __syncwarp();
              tmem_st8(t_o + dc, v);
              tmem_st8(t_o + dc + 8, v + 8);
            }
            tmem_wait_st();
          }
          const unsigned long long corr2 = pk2(corr, corr), vs2 = pk2(vs, vs);
#pragma unroll
          for (int dc = 0; dc < HD; dc += 32) {
            uint32_t v[32];
            tmem_ld32(t_o + dc, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const unsigned long long t = pk2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
              if constexpr (ES == 4)
                o2[dc / 2 + i] = fma2(t, vs2, mul2(o2[dc / 2 + i], corr2));
              else
                o2[dc / 2 + i] = fma2(o2[dc / 2 + i], corr2, t);
            }
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
      // the other group has read its tile outputs of this segment (every
      // product is complete then, and its warps are past the exchange of the
      // segment before)
      theirs += (n + w) / 2;
      if (theirs > 0)
        ok = __all_sync(0xffffffffu, chunk_wait(&sh->o_free[w ^ 1], (theirs - 1) & 1, sh, a, 52));
      if (!ok) break;
      if (warp_live) {
        sh->ml[w][row][0] = m;
        sh->ml[w][row][1] = l;
#pragma unroll
        for (int dc = 0; dc < HH; dc += 16) {
          uint32_t u[16];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 x = upk2(w == 0 ? o2[(HH + dc) / 2 + i] : o2[dc / 2 + i]);
            u[2 * i] = __float_as_uint(x.x);
            u[2 * i + 1] = __float_as_uint(x.y);
          }
          tmem_st16(t_mine + dc, u);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->xchg);
      ok = __all_sync(0xffffffffu, chunk_wait(&sh->xchg, seg & 1, sh, a, 51));
      if (!ok) break;
      tc_fence_after();
      const bool split = c.j0 > 0 || c.j1 < c.nk;
      const bool bad = *(volatile int*)&sh->bad[seg & 15] == seg + 1;
      // a piece that begins its row tile goes to the CTA's second place
      const size_t place = 2 * (size_t)blockIdx.x + (c.j0 == 0 ? 1 : 0);
      if (warp_live) {
        const long long row0 = (long long)c.q.q0 + c.rt * tt;
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
            tmem_ld16(t_theirs + dc + e, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 x =
                  upk2(w == 0 ? o2[(dc + e) / 2 + i] : o2[(HH + dc + e) / 2 + i]);
              tb[lane * 33 + e + 2 * i] = fmaf(__uint_as_float(v[2 * i]), f2, x.x * f) * inv;
              tb[lane * 33 + e + 2 * i + 1] = fmaf(__uint_as_float(v[2 * i + 1]), f2, x.y * f) * inv;
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
        long long ctas = (sum + chunk_min_tiles(BN) - 1) / chunk_min_tiles(BN);
        if (ctas > (long long)gridDim.x) ctas = gridDim.x;
        int* d = a.split + blockIdx.x * 8;
        d[0] = live_rows;
        d[1] = chunk_owner(c.unit, sum, (int)ctas);
        d[2] = c.s;
        d[3] = c.kvh;
        d[4] = c.rt;
      }
      __syncwarp();
      if (lane == 0) more = chunk_next<BN>(a, sh, c);
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
