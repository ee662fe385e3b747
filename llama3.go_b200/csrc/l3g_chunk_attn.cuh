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
// What bounds it (B200, 32 query and 8 kv heads of size 128).  f16 caches: the
// tensor core needs 2048 cycles for a tile's two times two products, half its
// rate for the one that a plain f16 attention takes, and the tiles follow each
// other at 2700 to 3400, the time that two alternating tiles need for scores,
// weights and output; 8 chunks of 1000 tokens after 7000: 2.1 to 2.3 ms, 430 to
// 470 TFLOP/s at the 1.35 to 1.5 GHz that the power limit leaves (each row tile
// reads its cache anew: 6.4 GB from memory, 42% of its rate).  64 decode
// steps after 512 to 8192: 300 to 320 us, 4.0 to 4.2 TB/s; of a tile's 128 rows 4
// are used, and one of the four schedulers does all of its exponentials.  f32
// caches: the loaders' conversion, 5000 cycles per tile and warp; 24 ragged
// sessions 188 to 196 us.  Short calls: the chain of latencies of a row tile, about
// 10000 cycles (8 us) to its first output; one token 22 us.
//
// Precision.  q, out and the statistics are fp32; the products run on the f16
// tensor cores.  An fp32 operand x goes in as two f16 terms, hi = f16(x) and
// lo = f16(x - hi), after scaling by a power of two (exact, undone in fp32), so
// it keeps 22 bits: q scaled per row, the weights p by 2^13 (taken out again where
// a tile's output joins the sums), the K and V tiles of an f32 cache per tile; f16
// caches go in as they are.  An f16 cache takes two products per tile (hi K,
// lo K), an f32 cache three (the lo lo term is below 2^-22).  The accumulators of one tile are fp32 in tensor memory; the
// sum over tiles is fp32 in registers, rounded to nearest, because the tensor
// core's own accumulation truncates and a long cache would add that up.
#pragma once

constexpr int CHUNK_BM = 128;       // rows per tile: lanes of tensor memory
// keys per tile (divides KV_PAGE): 128 of an f16 cache (64: 64 decode steps in
// 367 us instead of 316, 8 x 1000 tokens after 7000 in 2630 instead of 2300); 64
// of an f32 cache, whose tiles take twice the shared memory
__host__ __device__ constexpr int chunk_bn(int es) { return es == 2 ? 128 : 64; }
// warps: 16 softmax (four groups of four: group g is team g & 1, key half
// g >> 1), 4 output, 7 loaders, 1 that issues the products
constexpr int CHUNK_SOFT = 16;
constexpr int CHUNK_OUT = 4;
constexpr int CHUNK_LOAD = 7;
constexpr int CHUNK_WARP_OUT = CHUNK_SOFT;
constexpr int CHUNK_WARP_LOAD = CHUNK_WARP_OUT + CHUNK_OUT;
constexpr int CHUNK_WARP_MMA = CHUNK_WARP_LOAD + CHUNK_LOAD;
constexpr int CHUNK_WARPS = CHUNK_WARP_MMA + 1;
constexpr int CHUNK_THREADS = 32 * CHUNK_WARPS;
// registers per thread after the split; the block has 72 x 896 = 504 x 128.  An
// output thread holds HD of them.  The loaders of an f32 cache convert its
// tiles, and its softmax threads have half as many keys
__host__ __device__ constexpr int chunk_r_out(int hd) { return hd == 128 ? 168 : 104; }
__host__ __device__ constexpr int chunk_r_soft(int es) { return es == 2 ? 64 : 56; }
__host__ __device__ constexpr int chunk_r_rest(int hd, int es) {  // below the 72 of the launch
  return hd == 128 ? (504 - 168 - 4 * chunk_r_soft(es)) / 2 : 64;
}
static_assert(4 * chunk_r_soft(2) + chunk_r_out(64) + 2 * chunk_r_rest(64, 2) <= 504 &&
                  4 * chunk_r_soft(2) + chunk_r_out(128) + 2 * chunk_r_rest(128, 2) <= 504 &&
                  4 * chunk_r_soft(4) + chunk_r_out(128) + 2 * chunk_r_rest(128, 4) <= 504,
              "register split");
// keys a CTA takes at least (one token after 300, f32: 128 keys 21.9 us, 256 keys
// 22.4, 512 keys 26.6; long calls have more for each)
constexpr int CHUNK_MIN_KEYS = 128;
// what it costs to begin a row tile, in key tiles: q's terms, the first scores
// and the last output, 10000 to 14000 cycles, where a tile takes 3000 to 4000.
// (Ranges of equal tiles left SMs idle 40% of the time of 24 ragged sessions.
// Weight 1 / 4 / 6: 24 ragged f32 sessions 216 / 193 / 194 us, 64 decode steps
// 350 / 322 / 316, 7 x 300 tokens 44.8 / 45.0 / 43.3.)
constexpr int CHUNK_OPEN = 6;
__host__ __device__ constexpr int chunk_min_tiles(int bn) { return CHUNK_MIN_KEYS / bn; }
// the weights' scale, 2^13, and its inverse
constexpr float CHUNK_P_EXP = 13.0f, CHUNK_P_UP = 8192.0f, CHUNK_P_DOWN = 1.0f / 8192.0f;
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
  int ginv;          // row / group = row * ginv >> 16 for the rows of a tile
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
  long long unit;       // where its row tile begins in the linear order
  int s, kvh, rt, seg;
  int tiles;            // of the segments before
  l3g_chunk_seq q;      // the sequence's descriptor
  int nk, j0, j1;
};

struct ChunkSmem {
  uint8_t map[CHUNK_LOAD][128];  // (at the start: 128-byte aligned)
  uint64_t empty[CHUNK_LOAD], raw[CHUNK_LOAD];  // K / V slots
  // of tile t, at t & 7: its K tile is there and the weights that lie over its S
  // are spent; its V tile and weights are there and the output before is read
  uint64_t s_go[8], o_go[8];
  uint64_t s_full[2], o_full;
  uint64_t q_ready, l_full, e_done, drain;
  // per quarter of the rows: its four groups met, its team's two met
  uint64_t qx[4], mx[2][4];
  uint32_t tmem_base;
  int abort_flag;
  int alive;                     // changes while rows are taken again: nothing hangs
  int pad;
  long long begin, end;          // the CTA's range of the linear order
  long long unit0;               // where the row tile that holds `begin` begins
  int s0, kvh0, rt0, pad0;
  l3g_chunk_seq q0;              // its sequence's descriptor
  int bad[16];                   // segment + 1 whose pages are out of bounds
  float scale[32];               // f32 caches: 2^e of the items' tiles, item & 31
  ChunkCursor cur[CHUNK_WARPS];  // the warps' cursors, out of their registers
  float qmax[4][CHUNK_BM];       // largest |q| of each group's dims
  float gmax[2][2][2][CHUNK_BM]; // a tile's maxima [team][tile][key half]
  float m_tile[4][CHUNK_BM];     // what a tile's weights are relative to
  float m_team[2][CHUNK_BM], l_group[4][CHUNK_BM];  // a segment's statistics
  long long pre[L3G_CHUNK_SEQS_MAX + 1];  // where each sequence begins in the linear order
};
constexpr int CHUNK_HEAD = 23 * 1024;
static_assert(sizeof(ChunkSmem) <= CHUNK_HEAD, "chunk attention smem head");
// transposition buffers of a softmax and of an output warp: rows of 16 floats
constexpr int CHUNK_TBUF = 32 * 17 * 4, CHUNK_OBUF = 32 * 20 * 4;
__host__ __device__ constexpr int chunk_slot_bytes(int hd, int es) {
  return chunk_bn(es) * hd * es;  // f16: one operand tile; f32: its hi and lo tiles
}
// one slot per loader warp, as far as they fit
__host__ __device__ constexpr int chunk_slots(int hd, int es) {
  return (160 * 1024) / chunk_slot_bytes(hd, es) < CHUNK_LOAD
             ? (160 * 1024) / chunk_slot_bytes(hd, es)
             : CHUNK_LOAD;
}
__host__ __device__ constexpr int chunk_ring_off() {
  return (CHUNK_HEAD + CHUNK_SOFT * CHUNK_TBUF + CHUNK_OUT * CHUNK_OBUF + 1023) / 1024 * 1024;
}
// Operand tiles in shared memory: panels of up to 64 dims, [key][row bytes] with
// the 16-byte pieces of a row swizzled by the key (the tensor core's 128-byte
// and 64-byte swizzles), keys in groups of 8 one after another.  An f32 cache's
// panel is fetched as two raw panels of 32 floats, and each key's two raw rows
// become its hi and lo rows in place; with 32 dims a row holds hi, then lo.  The
// lane that converts piece c of both raw rows, dims 4 c and 32 + 4 c on, leaves
// them as piece c of the hi and the lo row: it overwrites only what it read, and
// no lane waits for another.  So 64 dims of an f32 tile lie in the order of
// chunk_dim, and so do q's, and the columns of the output.
__host__ __device__ constexpr int chunk_row_bytes(int hd, int es) {
  return es == 2 && hd < 64 ? 64 : 128;
}
__host__ __device__ constexpr int chunk_box_cols(int hd, int es) {  // elements of a box's row
  return es == 4 ? 32 : hd < 64 ? 32 : 64;
}
// the dim at place `at` of an operand row
__host__ __device__ constexpr int chunk_dim(int hd, int es, int at) {
  return es == 2 || hd < 64 ? at : (at & ~63) + (at >> 2 & 1) * 32 + (at >> 3 & 7) * 4 + (at & 3);
}
// byte of 16-byte piece `piece` of key k in a panel of rows of rb bytes
__host__ __device__ constexpr int chunk_piece(int rb, int k, int piece) {
  return k * rb + ((piece ^ (rb == 128 ? k & 7 : (k >> 1) & 3)) << 4);
}
__host__ __device__ constexpr int chunk_smem_bytes(int hd, int es) {
  return chunk_ring_off() + chunk_slots(hd, es) * chunk_slot_bytes(hd, es);
}

// Bounded wait of a whole warp, for waits that are on the critical path many
// times: no divergence, the warp suspended by the hardware (polling warps
// would take issue slots from the others) for 20 us a try, and the timer, which
// takes longer to read than most of the waits, looked at every 16th try.  The
// bound counts from the last sign of chunk_rows_again, which is longer at work
// the longer the cache is.
__device__ __forceinline__ bool chunk_wait(uint64_t* b, uint32_t parity, ChunkSmem* sh,
                                           const ChunkArgs& a, int where) {
  uint64_t t0 = 0;
  int alive = 0;
  for (int i = 0;; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(b, parity, 20000))) return true;
    if (__any_sync(0xffffffffu, *(volatile int*)&sh->abort_flag)) return false;
    if ((i & 15) == 15) {
      const uint64_t t = gtime();
      const int sign = *(volatile int*)&sh->alive;
      if (t0 == 0 || sign != alive) t0 = t;
      alive = sign;
      if (__any_sync(0xffffffffu, t - t0 > a.wait_ns)) {
        *(volatile int*)&sh->abort_flag = 1;
        if ((threadIdx.x & 31) == 0) report(a.res, ERR_TIMEOUT, where);
        return false;
      }
    }
  }
}

// Whether a descriptor stays inside its bounds (its pages are checked where
// they are read).
__device__ __forceinline__ bool chunk_seq_ok(const l3g_chunk_seq& s, int total_q) {
  // (a tensor copy needs a 16-byte aligned base)
  return s.pool && s.pages && ((uintptr_t)s.pool & 15) == 0 && ((uintptr_t)s.pages & 3) == 0 &&
         s.pps >= 0 && s.q0 >= 0 && s.n_q >= 0 && s.n_q <= total_q &&
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

// t * b / n for the ranges of the linear order (64-bit divisions take long)
__device__ __forceinline__ long long chunk_cut(long long t, int b, int n) {
  return t < 1 << 21 && n < 1 << 10 ? (long long)((uint32_t)t * (uint32_t)b / (uint32_t)n)
                                    : t * b / n;
}
// The CTAs share the linear order (sequence, kv head, row tile, key tile), in
// which a row tile has CHUNK_OPEN places before its key tiles, in equal ranges;
// a row tile whose keys several CTAs hold is joined by k_chunk_merge.  A cursor
// walks a CTA's range in segments, each the key tiles [j0, j1) of one row tile.
template <int BN>
__device__ __forceinline__ bool chunk_open(const ChunkArgs& a, const ChunkSmem* sh,
                                           ChunkCursor& c) {
  c.nk = chunk_tiles<BN>(c.q, CHUNK_BM / a.group, c.rt);
  const long long first = c.unit + CHUNK_OPEN, b = sh->begin - first, e = sh->end - first;
  c.j0 = b > 0 ? (int)b : 0;
  c.j1 = e < c.nk ? (int)e : c.nk;
  return c.j1 > c.j0;
}
template <int BN>
__device__ __forceinline__ bool chunk_first(const ChunkArgs& a, const ChunkSmem* sh,
                                            ChunkCursor& c) {
  if (sh->begin >= sh->end) return false;
  c.unit = sh->unit0;
  c.s = sh->s0;
  c.kvh = sh->kvh0;
  c.rt = sh->rt0;
  c.seg = 0;
  c.tiles = 0;
  c.q = sh->q0;
  return chunk_open<BN>(a, sh, c);
}
template <int BN>
__device__ __forceinline__ bool chunk_next(const ChunkArgs& a, const ChunkSmem* sh,
                                           ChunkCursor& c) {
  c.unit += CHUNK_OPEN + c.nk;
  if (c.unit + CHUNK_OPEN >= sh->end) return false;  // the next key tile is not in the range
  ++c.seg;
  c.tiles += c.j1 - c.j0;
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
  return chunk_open<BN>(a, sh, c);
}
// CTAs that take part, of an order of `sum` places
template <int BN>
__device__ __forceinline__ int chunk_ctas(long long sum) {
  constexpr int least = chunk_min_tiles(BN) + CHUNK_OPEN;
  return sum > (long long)gridDim.x * least ? (int)gridDim.x : (int)((sum + least - 1) / least);
}

// Warp 0: the places of every sequence in the order, then this CTA's range and where it starts.
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
        for (int rt = 0; rt < (q.n_q + tt - 1) / tt; ++rt)
          n += CHUNK_OPEN + chunk_tiles<BN>(q, tt, rt);
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
    const int ctas = chunk_ctas<BN>(sum);
    sh->begin = sh->end = 0;
    if ((int)blockIdx.x < ctas) {
      sh->begin = chunk_cut(sum, blockIdx.x, ctas);
      sh->end = chunk_cut(sum, blockIdx.x + 1, ctas);
      int lo = 0, hi = a.n_seqs - 1;  // the last sequence that starts at or before it
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (sh->pre[mid] <= sh->begin) lo = mid;
        else hi = mid - 1;
      }
      const l3g_chunk_seq q = a.seqs[lo];
      long long unit = sh->pre[lo];
      const long long all = sh->pre[lo + 1] - unit;  // a kv head's part of the sequence
      const long long per = chunk_cut(all, 1, a.hkv);
      const int kvh = all < 1 << 21 ? (int)((uint32_t)(sh->begin - unit) / (uint32_t)per)
                                    : (int)((sh->begin - unit) / per);
      unit += per * kvh;
      int rt = 0;
      for (;; ++rt) {
        const int n = CHUNK_OPEN + chunk_tiles<BN>(q, tt, rt);
        if (sh->begin < unit + n) break;
        unit += n;
      }
      sh->q0 = q;
      sh->s0 = lo;
      sh->kvh0 = kvh;
      sh->rt0 = rt;
      sh->unit0 = unit;
    }
  }
}

// The CTA whose range holds place t.
__device__ __forceinline__ int chunk_owner(long long t, long long sum, int ctas) {
  int c = (int)(t * ctas / sum);
  while (c + 1 < ctas && chunk_cut(sum, c + 1, ctas) <= t) ++c;
  while (c > 0 && chunk_cut(sum, c, ctas) > t) --c;
  return c;
}

// o[d] = sum_j p_j V_j[dim at place d0 + d], d < 16, over the n keys of `rows` that a row
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
    const float p = ex2(fmaf(s, scale, m == -INFINITY ? 0.0f : -m));
#pragma unroll 1
    for (int d = 0; d < 16; ++d)
      o[d] = fmaf(p, (float)k[HD + chunk_dim(HD, (int)sizeof(KT), d0 + d)], o[d]);
  }
}

// N words to N columns of the warp's lanes of tensor memory
template <int N>
__device__ __forceinline__ void tmem_stn(uint32_t t, const uint32_t* v) {
  if constexpr (N == 16) tmem_st16(t, v);
  else if constexpr (N == 8) tmem_st8(t, v);
  else tmem_st4(t, v);
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// The rows of a quarter (bits of `rows`, a lane each) whose sum over the segment
// came out as NaN, once more in fp32 from the cache itself, by the whole warp: a
// lane a key for the scores, HD / 32 dims a lane for the output.  An infinity of
// K comes as NaN from two-term operands (its lo term, or a q term that is zero
// or has the other sign), where a score of -inf weighs nothing.  A row with a
// score that is NaN or +inf, or with a q that is not finite, stays NaN, as it
// was written.  It hardly ever runs and is not made to be fast: one such key that
// all rows of 600 tokens see after 131072 positions (32 query and 8 kv heads of
// 128) costs 0.55 s, f32 1.3 s, where the call takes 2.4 and 5.1 ms.  The other
// warps' waits last that long, so it shows them that it is at work (alive).
template <int HD, typename KT>
__device__ __forceinline__ void chunk_rows_again(const ChunkArgs& a, const ChunkCursor& c,
                                                 uint32_t rows, int quarter, int lane, bool split,
                                                 size_t place, int* alive) {
  constexpr int V = HD / 32, BN = chunk_bn((int)sizeof(KT)), W = 16 / (int)sizeof(KT);
  struct alignas(16) Piece {
    KT x[W];
  };
  struct alignas(V * sizeof(KT)) Dims {
    KT x[V];
  };
  const int tt = CHUNK_BM / a.group;
  const int* pages = c.q.pages + ((size_t)a.layer * a.hkv + c.kvh) * c.q.pps;
  // the keys from kb on, up to the page's end; null for a page outside its pool
  auto cells_at = [&](int kb) -> const KT* {
    if ((kb & (KV_PAGE - 1)) == 0 && lane == 0) ++*(volatile int*)alive;
    const int page = pages[kb / KV_PAGE];
    if (page < 0 || page >= c.q.n_pages) return nullptr;
    return reinterpret_cast<const KT*>(c.q.pool) +
           ((size_t)page * KV_PAGE + (kb & (KV_PAGE - 1))) * 2 * HD;
  };
  auto q_at = [&](int row) {
    const int tok = row * a.ginv >> 16;
    return a.q + ((long long)c.q.q0 + (long long)c.rt * tt + tok) * a.ldq +
           (size_t)(c.kvh * a.group + row - tok * a.group) * HD;
  };
  // rows with a finite q, and the first keys with a NaN and with an infinity:
  // a row that sees the one stays NaN, one that does not see the other too
  uint32_t left = 0;
#pragma unroll 1
  for (; rows; rows &= rows - 1) {
    const float* q = q_at(quarter * 32 + __ffs(rows) - 1) + lane * V;
    bool good = true;
#pragma unroll
    for (int i = 0; i < V; ++i) good = good && fabsf(q[i]) <= 3.4028235e38f;
    if (__all_sync(0xffffffffu, good)) left |= rows & (0u - rows);
  }
  const int last = min(c.j1 * BN, c.q.kv_len);
  int nan_at = last, inf_at = last;
#pragma unroll 1
  for (int kb = c.j0 * BN; kb < last && left && nan_at == last; kb += 32) {  // (32 divides a page)
    const KT* cells = cells_at(kb);
    if (!cells) return;
    bool nan = false, inf = false;
    if (kb + lane < last) {
#pragma unroll 4
      for (int d = 0; d < HD; d += W) {
        const Piece x = *reinterpret_cast<const Piece*>(cells + (size_t)lane * 2 * HD + d);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float f = (float)x.x[i];
          nan = nan || f != f;
          inf = inf || fabsf(f) > 3.4028235e38f;
        }
      }
    }
    const uint32_t bn = __ballot_sync(0xffffffffu, nan), bi = __ballot_sync(0xffffffffu, inf);
    if (bn) nan_at = kb + __ffs(bn) - 1;
    if (bi && inf_at == last) inf_at = kb + __ffs(bi) - 1;
  }
#pragma unroll 1
  for (; left; left &= left - 1) {
    const int row = quarter * 32 + __ffs(left) - 1, tok = row * a.ginv >> 16;
    const long long at = (long long)c.q.q0 + (long long)c.rt * tt + tok;
    const int head = c.kvh * a.group + row - tok * a.group;
    const float* q = q_at(row);
    const int end = min(c.j1 * BN, c.q.kv_len - c.q.n_q + c.rt * tt + tok + 1);
    if (end > nan_at || end <= inf_at) continue;
    float M = -INFINITY, L = 0.0f, o[V];
    bool good = true;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.0f;
#pragma unroll 1
    for (int kb = c.j0 * BN; kb < end && good; kb += 32) {
      const int cnt = min(32, end - kb);
      const KT* cells = cells_at(kb);
      float s = -INFINITY;
      if (lane < cnt) {
        const KT* k = cells + (size_t)lane * 2 * HD;
        float d4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int d = 0; d < HD; d += W) {
          const Piece x = *reinterpret_cast<const Piece*>(k + d);
#pragma unroll
          for (int i = 0; i < W; i += 4) {
            const float4 y = *reinterpret_cast<const float4*>(q + d + i);
            d4[0] = fmaf(y.x, (float)x.x[i], d4[0]);
            d4[1] = fmaf(y.y, (float)x.x[i + 1], d4[1]);
            d4[2] = fmaf(y.z, (float)x.x[i + 2], d4[2]);
            d4[3] = fmaf(y.w, (float)x.x[i + 3], d4[3]);
          }
        }
        s = ((d4[0] + d4[1]) + (d4[2] + d4[3])) * a.scale;
      }
      good = __all_sync(0xffffffffu, s < INFINITY);
      if (!good) break;
      const float mn = fmaxf(M, warp_max(s)), mu = mn == -INFINITY ? 0.0f : mn;
      const float f = M == -INFINITY ? 0.0f : ex2(M - mu);
      const float p = ex2(s - mu);
      L = fmaf(L, f, warp_sum(p));
      M = mn;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] *= f;
#pragma unroll 8
      for (int j = 0; j < cnt; ++j) {
        const float pj = __shfl_sync(0xffffffffu, p, j);
        const Dims v = *reinterpret_cast<const Dims*>(cells + (size_t)j * 2 * HD + HD + lane * V);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = fmaf(pj, (float)v.x[i], o[i]);
      }
    }
    if (!good) continue;
    float* to = split ? a.part_o + (place * CHUNK_BM + row) * HD
                      : a.out + at * a.ldo + (size_t)head * HD;
    const float inv = split ? 1.0f : L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
#pragma unroll
    for (int i = 0; i < V; ++i) to[lane * V + i] = o[i] * inv;
    if (split && lane == 0) {
      a.part_ml[(place * CHUNK_BM + row) * 2] = M;
      a.part_ml[(place * CHUNK_BM + row) * 2 + 1] = L;
    }
  }
}

// 2^e as a float, e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// the exponent of the largest magnitude m, limited so that pow2i takes the
// scale factors that come from it; NaN and infinity count as the largest
__device__ __forceinline__ int exp_of(float m) {
  const int e = (__float_as_int(m) >> 23 & 255) - 127;
  return e < -100 ? -100 : e > 127 ? 127 : e;
}

// Roles.  One warp issues the products, in the order S0 S1 O0 S2 O1 ...:
//   S = q K^T   A = q from tensor memory, B = K tile  [key][dim], K-major
//   O = p V     A = p from tensor memory (over S), B = V tile [key][dim], MN-major
// Seven loader warps bring the tiles into a ring of shared-memory slots in that
// order.  Sixteen softmax warps turn scores into weights: two teams take the
// tiles in turn (there are two S), a thread a row and half of the tile's keys;
// each team has a running maximum of its own.  Four output warps, a thread a
// row, add a tile's output, scaled to the maximum over both teams, to the
// registers that hold the row's.  The tensor core waits for the weights of tile
// j only after it has been given the scores of tile j + 1.
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
  pdl_launch_dependents();

  if (threadIdx.x == 32 * CHUNK_WARP_LOAD) {  // (while warp 0 plans)
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh->empty[i], 1);
      mbar_init(&sh->raw[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&sh->qx[i], 4);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh->s_full[w], 1);
      for (int i = 0; i < 4; ++i) mbar_init(&sh->mx[w][i], 2);
    }
    for (int i = 0; i < 8; ++i) {
      mbar_init(&sh->s_go[i], 2);
      mbar_init(&sh->o_go[i], 1 + CHUNK_SOFT / 2 + CHUNK_OUT);
    }
    mbar_init(&sh->o_full, 1);
    mbar_init(&sh->q_ready, CHUNK_SOFT);
    mbar_init(&sh->l_full, CHUNK_SOFT);
    mbar_init(&sh->e_done, CHUNK_OUT);
    mbar_init(&sh->drain, 1);
    sh->abort_flag = sh->alive = 0;
    for (int i = 0; i < 16; ++i) sh->bad[i] = 0;
    fence_mbar_init();
    mbar_arrive(&sh->s_go[0]);  // nothing lies over the first two S
    mbar_arrive(&sh->s_go[1]);
  }
  if (warp == 0) {
    chunk_plan<BN>(a, sh, lane);
  }
  if (warp == CHUNK_WARP_MMA) tmem_alloc(&sh->tmem_base, CHUNK_T_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;

  // every warp walks the CTA's segments with a cursor of its own: lane 0 moves
  // it between two __syncwarp, which order the lanes' reads of the old segment
  // before the write and those of the new one behind it (a shuffle orders
  // registers, not memory)
  ChunkCursor& c = sh->cur[warp];
  auto first = [&] {
    bool more = false;
    if (lane == 0) more = chunk_first<BN>(a, sh, c);
    __syncwarp();
    return __shfl_sync(0xffffffffu, more ? 1 : 0, 0) != 0;
  };
  auto next = [&] {
    bool more = false;
    __syncwarp();
    if (lane == 0) more = chunk_next<BN>(a, sh, c);
    __syncwarp();
    return __shfl_sync(0xffffffffu, more ? 1 : 0, 0) != 0;
  };
  auto wait = [&](uint64_t* b, int phase, int site) {
    return chunk_wait(b, phase & 1, sh, a, site);
  };
  const int quarter = warp & 3;          // softmax and output warps: their rows
  const int row = quarter * 32 + lane;
  const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
  bool ok = true;

  if (warp >= CHUNK_WARP_LOAD) {
  regs_dec<chunk_r_rest(HD, ES)>();
  if (warp < CHUNK_WARP_MMA) {
    // ---- loaders ----------------------------------------------------------
    // Warp lw brings the items lw, lw + NS, ... whole into slot lw: a tile whose
    // keys all exist by tensor copies (one box per panel), the last, part-filled
    // one by 16-byte copies with zeros for the keys past the cache's end.
    const int lw = warp - CHUNK_WARP_LOAD;
    const int kl = lane >> 3, cl = lane & 7;  // key and piece of the lane
    uint8_t* map = a.maps + ((size_t)blockIdx.x * CHUNK_LOAD + lw) * 128;
    const void* map_pool = nullptr;
    uint8_t* const dst = ring + (size_t)lw * SLOT;
    int it = lw;                  // this warp's next item
    int it0 = 0;                  // the segment's first
    ok = lw < NS;
    for (bool more = ok && first(); more && ok; more = next()) {
      {  // the segment's q rows into L2, ahead of the softmax warps' loads
        const int live_rows = min(tt, c.q.n_q - c.rt * tt) * a.group;
        const float* q0 = a.q + ((long long)c.q.q0 + (long long)c.rt * tt) * a.ldq +
                          (size_t)c.kvh * a.group * HD;
        constexpr int LINES = HD / 32;  // of 128 bytes per row
        for (int e = lw * 32 + lane; e < live_rows * LINES; e += NS * 32) {
          const int r = e / LINES, tok = r * a.ginv >> 16;
          prefetch_l2(q0 + tok * a.ldq + (r - tok * a.group) * HD + e % LINES * 32);
        }
      }
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
          ok = chunk_wait(&sh->empty[lw], (use - 1) & 1, sh, a, 40);
          if (!ok) break;
        }
        // (after the wait: the slot's last copy, which used the map, is over)
        if (cnt == BN && map_pool != c.q.pool) {
          map_pool = c.q.pool;
          tmap_rebase(map, sh->map[lw], &a.map, map_pool, lane);
        }
        const int tile = (it0 >> 1) + j - c.j0;
        uint64_t* go = is_v ? &sh->o_go[tile & 7] : &sh->s_go[tile & 7];
        uint64_t* landed = ES == 2 ? go : &sh->raw[lw];
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
          ok = chunk_wait(&sh->raw[lw], use & 1, sh, a, 41);
          if (!ok) break;
          // the tile's scale, from its largest finite magnitude (a NaN loses
          // against every number)
          float m = 0.0f, m1 = 0.0f;
#pragma unroll 1
          for (int e = lane; e < SLOT / 16; e += 256) {
            float4 x[8];
#pragma unroll
            for (int i2 = 0; i2 < 8; ++i2)
              x[i2] = reinterpret_cast<const float4*>(dst)[e + 32 * i2];
#pragma unroll
            for (int i2 = 0; i2 < 8; ++i2) {
              m = max3(m, fabsf(x[i2].x), fabsf(x[i2].y));
              m1 = max3(m1, fabsf(x[i2].z), fabsf(x[i2].w));
            }
          }
          m = warp_max(fmaxf(m, m1));
          if (m > 3.4028235e38f) {
            m = 0.0f;
#pragma unroll 1
            for (int e = lane; e < SLOT / 4; e += 32) {
              const float v = fabsf(reinterpret_cast<const float*>(dst)[e]);
              if (v <= 3.4028235e38f) m = fmaxf(m, v);
            }
            m = warp_max(m);
          }
          const int e2 = exp_of(m);  // it lands in [2^14, 2^15)
          const float up = pow2i(14 - e2);
          if (lane == 0) sh->scale[it & 31] = 1.0f / up;
          const unsigned long long up2 = pk2(up, up), neg2 = pk2(-1.0f, -1.0f);
          // the two terms of four floats
          auto split = [&](const float4& x, uint2& hi, uint2& lo) {
            const unsigned long long f0 = mul2(pk2(x.x, x.y), up2);
            const unsigned long long f1 = mul2(pk2(x.z, x.w), up2);
            const float2 a0 = upk2(f0), a1 = upk2(f1);
            hi.x = pack_h2(a0.x, a0.y);
            hi.y = pack_h2(a1.x, a1.y);
            const float2 b0 = unpack_h2(hi.x), b1 = unpack_h2(hi.y);
            const float2 c0 = upk2(fma2(pk2(b0.x, b0.y), neg2, f0));
            const float2 c1 = upk2(fma2(pk2(b1.x, b1.y), neg2, f1));
            lo.x = pack_h2(c0.x, c0.y);
            lo.y = pack_h2(c1.x, c1.y);
          };
          if constexpr (HD >= 64) {
            // four keys' loads before the stores, which the compiler has to keep
            // in their order: a step that waits for its own loads takes 175 cycles
#pragma unroll 1
            for (int p = 0; p < PANELS; p += 2) {
              uint8_t* r0 = dst + p * BOX;
#pragma unroll 1
              for (int k0 = kl; k0 < BN; k0 += 16) {
                float4 x[4], y[4];
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2) {
                  const uint8_t* at = r0 + chunk_piece(128, k0 + 4 * i2, cl);
                  x[i2] = *reinterpret_cast<const float4*>(at);
                  y[i2] = *reinterpret_cast<const float4*>(at + BOX);
                }
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2) {
                  uint8_t* at = r0 + chunk_piece(128, k0 + 4 * i2, cl);
                  uint2 h0, h1, l0, l1;
                  split(x[i2], h0, l0);
                  split(y[i2], h1, l1);
                  *reinterpret_cast<uint4*>(at) = make_uint4(h0.x, h0.y, h1.x, h1.y);
                  *reinterpret_cast<uint4*>(at + BOX) = make_uint4(l0.x, l0.y, l1.x, l1.y);
                }
              }
            }
          } else {
#pragma unroll 1
            for (int k = kl; k < BN; k += 4) {
              const float4 x = *reinterpret_cast<const float4*>(dst + chunk_piece(128, k, cl));
              __syncwarp();
              uint2 hi, lo;
              split(x, hi, lo);
              *reinterpret_cast<uint2*>(dst + chunk_piece(128, k, cl >> 1) + (cl & 1) * 8) = hi;
              *reinterpret_cast<uint2*>(dst + chunk_piece(128, k, 4 + (cl >> 1)) + (cl & 1) * 8) = lo;
            }
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(go);
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
    // The whole warp walks the loop, one lane issues.  The tensor core takes new
    // products only while it has about four left (280 cycles), so a batch has
    // one barrier for all that it needs: a wait takes 100 to 200.
    int it = 0;          // slots used
    int ns = 0, no = 0;  // tiles so far, issued to S and to O
    for (bool more = first(); more && ok; more = next()) {
      const int n = __shfl_sync(0xffffffffu, c.j1 - c.j0, 0);
      ok = wait(&sh->q_ready, c.seg, 42);
      for (int j = 0; j <= n && ok; ++j) {
        if (j < n) {
          const int w = ns & 1, slot = it % NS;
          ok = wait(&sh->s_go[ns & 7], ns >> 3, 43);
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
          ++ns;
          ++it;
        }
        if (j >= 1) {
          const int w = no & 1, slot = it % NS;
          ok = wait(&sh->o_go[no & 7], no >> 3, 46);
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
            mma_commit(&sh->s_go[(no + 2) & 7]);
            mma_commit(&sh->o_full);
            mma_commit(&sh->empty[slot]);
          }
          __syncwarp();
          ++no;
          ++it;
        }
      }
    }
    if (ns > 0) {  // every product issued has completed before the memory goes
      if (elect_one()) mma_commit(&sh->drain);
      int dummy = 0;
      mbar_wait(&sh->drain, 0, &dummy, a.res, 48, a.wait_ns);
    }
    __syncwarp();
  }
  } else if (warp >= CHUNK_WARP_OUT) {
    // ---- output -------------------------------------------------------------
    regs_inc<chunk_r_out(HD)>();
    const uint32_t t_o = t_lane + CHUNK_T_O;
    float* tb = tbuf + CHUNK_SOFT * (CHUNK_TBUF / 4) + (warp - CHUNK_WARP_OUT) * (CHUNK_OBUF / 4);
    int done = 0;  // tiles so far
    // the next tile's product may overwrite the output: also from the start
    if (lane == 0) mbar_arrive(&sh->o_go[0]);
    if (warp == CHUNK_WARP_OUT && lane == 0) a.split[blockIdx.x * 8] = 0;
    for (bool more = first(); more; more = next()) {
      const int n = c.j1 - c.j0, seg = c.seg;
      const int live_rows = min(tt, c.q.n_q - c.rt * tt) * a.group;
      const bool warp_live = quarter * 32 < live_rows, live = row < live_rows;
      // keys from the segment's first on that the row sees
      const int seen0 =
          live ? c.q.kv_len - c.q.n_q + c.rt * tt + (row * a.ginv >> 16) + 1 - c.j0 * BN : 0;
      const int item0 = ES == 4 ? 2 * c.tiles : 0;
      unsigned long long o2[HD / 2];  // the output, dims 2 i and 2 i + 1
      float M = -INFINITY;            // what it is relative to
#pragma unroll
      for (int d = 0; d < HD / 2; ++d) o2[d] = 0ull;
      for (int j = 0; j < n; ++j, ++done) {
        ok = wait(&sh->o_full, done, 50);
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          const float mt = sh->m_tile[done & 3][row];
          float vs = 1.0f;  // (a loader is at most NS + 6 items ahead)
          if constexpr (ES == 4)
            vs = *(volatile float*)&sh->scale[(item0 + (j == n - 1 ? 2 * n - 1 : 2 * j + 2)) & 31];
          const int seen = min(max(seen0 - j * BN, 0), BN);
          if (!__all_sync(0xffffffffu, seen == BN || !live)) {
            bool odd = false;  // did an unseen NaN or infinity come in?
#pragma unroll 1
            for (int dc = 0; dc < HD; dc += 16) {
              uint32_t v[16];
              tmem_get16(t_o + dc, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) odd |= !(fabsf(__uint_as_float(v[i])) <= 3.4028235e38f);
            }
            odd = odd && live && seen < BN;
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
                tmem_get16(t_o + dc, v);
                if (odd) {
                  chunk_row_slow<HD, KT>(rows, in ? seen : 0, qrow, a.scale, mt, dc, tb + lane * 20);
#pragma unroll
                  for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(tb[lane * 20 + i] / vs * CHUNK_P_UP);
                }
                __syncwarp();
                tmem_st16(t_o + dc, v);
              }
              tmem_wait_st();
            }
          }
          const float mn = fmaxf(M, mt);
          const float co = M == -INFINITY ? 0.0f : ex2(M - mn);
          // (the weights' scale goes here, or finite outputs of an f32 cache's
          // largest values would pass fp32's range)
          const float ct = mt == -INFINITY ? 0.0f : ex2(mt - mn) * (vs * CHUNK_P_DOWN);
          M = mn;
          const unsigned long long co2 = pk2(co, co), ct2 = pk2(ct, ct);
          const bool same = __all_sync(0xffffffffu, co == 1.0f);
#pragma unroll
          for (int dc = 0; dc < HD; dc += 32) {
            uint32_t v[32];
            tmem_get32(t_o + dc, v);
            if (dc + 32 >= HD) {  // the next product may overwrite it
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh->o_go[(done + 1) & 7]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              unsigned long long& o = o2[dc / 2 + i];
              if (!same) o = mul2(o, co2);
              o = fma2(pk2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ct2, o);
            }
          }
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->o_go[(done + 1) & 7]);
        }
      }
      if (!ok) break;
      ok = wait(&sh->l_full, seg, 51);
      if (!ok) break;
      float L = 0.0f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float mg = sh->m_team[g & 1][row];
        L = fmaf(sh->l_group[g][row], mg == -INFINITY ? 0.0f : ex2(mg - M) * CHUNK_P_DOWN, L);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->e_done);
      const bool split = c.j0 > 0 || c.j1 < c.nk;
      const bool bad = *(volatile int*)&sh->bad[seg & 15] == seg + 1;
      // a piece that begins its row tile goes to the CTA's second place
      const size_t place = 2 * (size_t)blockIdx.x + (c.j0 == 0 ? 1 : 0);
      if (warp_live) {
        const long long row0 = (long long)c.q.q0 + c.rt * tt;
        const int head0 = c.kvh * a.group;
        const float inv = split ? 1.0f : L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
        if (split && live) {
          a.part_ml[(place * CHUNK_BM + row) * 2] = bad ? __int_as_float(0x7fc00000) : M;
          a.part_ml[(place * CHUNK_BM + row) * 2 + 1] = L;
        }
        // through shared memory, 16 dims at a time, four lanes a row; the next
        // segment's products wait for this, so all addresses are ready before
        // and the stores of a step do not wait for each other (128 rows x 128
        // dims in a rolled loop: 8000 to 14000 cycles)
        const int rl = lane >> 2, d4 = (lane & 3) * 4;
        float* to[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = quarter * 32 + i * 8 + rl, tok = r * a.ginv >> 16;
          to[i] = split ? a.part_o + (place * CHUNK_BM + r) * HD
                        : a.out + (row0 + tok) * a.ldo + (size_t)(head0 + r - tok * a.group) * HD;
          if (r >= live_rows || (bad && !split)) to[i] = nullptr;
        }
#pragma unroll
        for (int dc = 0; dc < HD; dc += 16) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = upk2(o2[dc / 2 + 2 * i]), y = upk2(o2[dc / 2 + 2 * i + 1]);
            *reinterpret_cast<float4*>(tb + lane * 20 + 4 * i) =
                make_float4(x.x * inv, x.y * inv, y.x * inv, y.y * inv);
          }
          __syncwarp();
          const int dim = chunk_dim(HD, ES, dc + d4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(tb + (i * 8 + rl) * 20 + d4);
            if (to[i]) *reinterpret_cast<float4*>(to[i] + dim) = x;
          }
        }
        const uint32_t again = __ballot_sync(0xffffffffu, live && !bad && L != L);
        if (again) {
          __syncwarp();  // (over what other lanes have written)
          chunk_rows_again<HD, KT>(a, c, again, quarter, lane, split, place, &sh->alive);
        }
      }
      if (warp == CHUNK_WARP_OUT && lane == 0 && split && c.j1 == c.nk) {
        // this CTA ends the row tile: what k_chunk_merge joins
        const long long sum = sh->pre[a.n_seqs];
        int* d = a.split + blockIdx.x * 8;
        d[0] = live_rows;
        d[1] = chunk_owner(c.unit + CHUNK_OPEN, sum, chunk_ctas<BN>(sum));
        d[2] = c.s;
        d[3] = c.kvh;
        d[4] = c.rt;
      }
    }
  } else {
    // ---- softmax ------------------------------------------------------------
    regs_dec<chunk_r_soft(ES)>();
    constexpr int KG = BN / 2;  // keys of a tile per thread
    constexpr int DG = HD / 4;  // dims of q per group
    const int g = warp >> 2, team = g & 1, half = g >> 1;
    const uint32_t t_s = t_lane + CHUNK_T_S + team * BN + half * KG;
    float* tb = tbuf + warp * 32 * 17;
    int t0 = 0;            // tiles of the segments before
    int qph = 0, mph = 0;  // phases of qx and mx
    for (bool more = first(); more; more = next()) {
      const int n = c.j1 - c.j0, seg = c.seg;
      const int live_rows = min(tt, c.q.n_q - c.rt * tt) * a.group;
      const bool warp_live = quarter * 32 < live_rows, live = row < live_rows;
      // keys from the segment's first on that the row sees
      const int seen0 =
          live ? c.q.kv_len - c.q.n_q + c.rt * tt + (row * a.ginv >> 16) + 1 - c.j0 * BN : 0;
      const int item0 = ES == 4 ? 2 * c.tiles : 0;
      // the last product that reads the q before this is complete
      if (t0 > 0) ok = wait(&sh->s_full[(t0 - 1) & 1], (t0 - 1) >> 1, 53);
      if (!ok) break;
      tc_fence_after();
      float sc = 0.0f;
      if (warp_live) {
        const long long row0 = (long long)c.q.q0 + c.rt * tt;
        const int head0 = c.kvh * a.group;
        // eight lanes read a row, four rows at a time, all in flight at once;
        // group g takes the places [g DG, g DG + DG); the terms go through shared
        // memory to one row per lane
        const int rl4 = lane >> 3, l8 = lane & 7;
        constexpr int VL = DG / 8;  // floats of a row per lane
        float x[8][VL];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = quarter * 32 + i * 4 + rl4;
          const int tok = r * a.ginv >> 16;
          const float* src = a.q + (row0 + tok) * a.ldq +
                             (size_t)(head0 + r - tok * a.group) * HD +
                             chunk_dim(HD, ES, g * DG + l8 * VL);
          if constexpr (VL == 4) {
            const float4 y = r < live_rows ? *reinterpret_cast<const float4*>(src)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
            x[i][0] = y.x, x[i][1] = y.y, x[i][2] = y.z, x[i][3] = y.w;
          } else {
#pragma unroll
            for (int k = 0; k < VL; ++k) x[i][k] = r < live_rows ? src[k] : 0.0f;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float m = 0.0f;
#pragma unroll
          for (int k = 0; k < VL; ++k) m = fmaxf(m, fabsf(x[i][k]));
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          if (l8 == 0) sh->qmax[g][quarter * 32 + i * 4 + rl4] = m;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->qx[quarter]);
        ok = wait(&sh->qx[quarter], qph++, 54);
        if (!ok) break;
        // a row's largest value lands in [2^10, 2^11)
        auto up_of = [&](int r) {
          return pow2i(10 - exp_of(fmaxf(fmaxf(sh->qmax[0][r], sh->qmax[1][r]),
                                         fmaxf(sh->qmax[2][r], sh->qmax[3][r]))));
        };
        sc = a.scale / up_of(row);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float up = up_of(quarter * 32 + i * 4 + rl4);
#pragma unroll
          for (int k = 0; k < VL; ++k) x[i][k] *= up;
        }
        uint32_t* tw = reinterpret_cast<uint32_t*>(tb);
        constexpr int W = DG / 2;  // packed words of a row's term, at most 16
#pragma unroll 1
        for (int term = 0; term < 2; ++term) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t* t = tw + (i * 4 + rl4) * 17;
            if constexpr (VL > 1) {
#pragma unroll
              for (int k = 0; k < VL; k += 2) {
                const float y0 = x[i][k], y1 = x[i][k + 1];
                uint32_t p = pack_h2(y0, y1);
                if (term == 1) {
                  const float2 b = unpack_h2(p);
                  p = pack_h2(y0 - b.x, y1 - b.y);
                }
                t[l8 * (VL / 2) + k / 2] = p;
              }
            } else {
              const float y = x[i][0];
              const __half h = __float2half_rn(y);
              reinterpret_cast<__half*>(t)[l8] =
                  term == 0 ? h : __float2half_rn(y - __half2float(h));
            }
          }
          __syncwarp();
          uint32_t u[W];
#pragma unroll
          for (int i = 0; i < W; ++i) u[i] = tw[lane * 17 + i];
          tmem_stn<W>(t_lane + CHUNK_T_Q + term * (HD / 2) + g * W, u);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->q_ready);

      float m = -INFINITY, l = 0.0f;  // the team's maximum, this thread's sum
      for (int j = (t0 ^ team) & 1; j < n; j += 2) {
        const int tile = t0 + j;
        ok = wait(&sh->s_full[team], tile >> 1, 49);
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          // this thread's keys of the tile that the row sees
          const int seen = min(max(seen0 - j * BN - half * KG, 0), KG);
          const bool whole = __all_sync(0xffffffffu, seen == KG || !live);
          float ks = sc;  // (a loader is at most NS + 6 items ahead)
          if constexpr (ES == 4)
            ks *= *(volatile float*)&sh->scale[(item0 + (j == 0 ? 0 : 2 * j - 1)) & 31];
          float mx = -INFINITY;
          if (whole) {
            float m2 = -INFINITY;
            uint32_t v[32];
#pragma unroll
            for (int h = 0; h < KG; h += 32) {
              tmem_get32(t_s + h, v);
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                mx = max3(mx, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                m2 = max3(m2, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
              }
            }
            mx = fmaxf(mx, m2);
          } else {
#pragma unroll 1
            for (int h = 0; h < KG; h += 16) {
              uint32_t v[16];
              tmem_get16(t_s + h, v);
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (h + i < seen) mx = fmaxf(mx, __uint_as_float(v[i]));
            }
          }
          // the row's other half of the keys
          const int gb = tile >> 1 & 1;
          sh->gmax[team][gb][half][row] = mx;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->mx[team][quarter]);
          ok = wait(&sh->mx[team][quarter], mph++, 55);
          if (!ok) break;
          mx = fmaxf(mx, sh->gmax[team][gb][half ^ 1][row]);
          const float mn = fmaxf(m, mx * ks);
          const float mu = mn == -INFINITY ? 0.0f : mn;
          l *= m == -INFINITY ? 0.0f : ex2(m - mu);
          m = mn;
          if (half == 0) sh->m_tile[tile & 3][row] = m;
          const float off = CHUNK_P_EXP - mu;
          const unsigned long long ks2 = pk2(ks, ks), off2 = pk2(off, off);
          const unsigned long long neg2 = pk2(-1.0f, -1.0f);
          unsigned long long sum = 0ull;  // a pair of fp32
          // weights of 16 keys from h on, over their scores; ALL: the row sees them
          auto weigh = [&](int h, auto all) {
            uint32_t v[16], ph[8], pl[8];
            tmem_get16(t_s + h, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 t = upk2(
                  fma2(pk2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ks2, off2));
              float x = ex2(t.x), y = ex2(t.y);
              if constexpr (!decltype(all)::value) {
                if (h + 2 * i >= seen) x = 0.0f;
                if (h + 2 * i + 1 >= seen) y = 0.0f;
              }
              const unsigned long long p2 = pk2(x, y);
              sum = add2(sum, p2);
              ph[i] = pack_h2(x, y);
              const float2 b = unpack_h2(ph[i]);
              const float2 r = upk2(fma2(pk2(b.x, b.y), neg2, p2));
              pl[i] = pack_h2(r.x, r.y);
            }
            tmem_st8(t_s + h, ph);
            tmem_st8(t_s + h + 8, pl);
          };
          if (whole) {
#pragma unroll 1
            for (int h = 0; h < KG; h += 16) weigh(h, std::true_type());
          } else {
#pragma unroll 1
            for (int h = 0; h < KG; h += 16) weigh(h, std::false_type());
          }
          const float2 total = upk2(sum);
          l += total.x + total.y;
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->o_go[tile & 7]);
      }
      if (!ok) break;
      t0 += n;
      // the statistics, once those of the segment before have been read
      if (seg > 0) ok = wait(&sh->e_done, seg - 1, 52);
      if (!ok) break;
      sh->l_group[g][row] = l;
      if (half == 0) sh->m_team[team][row] = m;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->l_full);
    }
  }
  cp_async_wait<0>();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == CHUNK_WARP_MMA) {
    __syncwarp();
    tmem_dealloc(tmem, CHUNK_T_COLS);
  }
}

// Joins the pieces of a row tile that several CTAs hold, in the order of the
// CTAs: out = sum O_p 2^(m_p - M) / sum l_p 2^(m_p - M).  grid (CTAs of the
// attention, CHUNK_BM / 8), 256 threads, a warp a row: its lanes take the
// pieces' statistics side by side, then it adds the outputs, whose loads do not
// wait for each other.  (A block a row at a time, with barriers, took 28 us for
// 148 row tiles of two pieces.)  Launched early: it waits for the pieces itself.
template <int HD>
__global__ void __launch_bounds__(256) k_chunk_merge(const __grid_constant__ ChunkArgs a) {
  pdl_wait();
  const int* d = a.split + blockIdx.x * 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y * 8 + warp;
  if (r >= d[0]) return;  // (0: no split row tile ends in this CTA)
  const int c0 = d[1], n = (int)blockIdx.x - c0 + 1;
  const l3g_chunk_seq q = a.seqs[d[2]];
  const int tt = CHUNK_BM / a.group;
  constexpr int V = HD / 32;
  float M = -INFINITY, L = 0.0f, o[V];
  bool bad = false;  // a maximum that is NaN marks a piece with a page outside its pool
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.0f;
  // (a piece that begins its row tile lies in its CTA's second place)
  auto place = [&](int p) { return (2 * (size_t)(c0 + p) + (p == 0 ? 1 : 0)) * CHUNK_BM + r; };
  for (int p0 = 0; p0 < n; p0 += 32) {
    const int cnt = min(32, n - p0);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < cnt) ml = *reinterpret_cast<const float2*>(a.part_ml + place(p0 + lane) * 2);
    bad = bad || __any_sync(0xffffffffu, ml.x != ml.x);
    const float mn = fmaxf(M, warp_max(ml.x));
    const float f = M == -INFINITY ? 0.0f : ex2(M - mn);
    const float g = ml.x == -INFINITY ? 0.0f : ex2(ml.x - mn);
    M = mn;
    L = fmaf(L, f, warp_sum(ml.y * g));
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] *= f;
#pragma unroll 4
    for (int p = 0; p < cnt; ++p) {
      const float gp = __shfl_sync(0xffffffffu, g, p);
      const float* po = a.part_o + place(p0 + p) * HD;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(po[i * 32 + lane], gp, o[i]);
    }
  }
  if (bad) return;
  float* out = a.out + ((long long)q.q0 + (long long)d[4] * tt + r / a.group) * a.ldo +
               (size_t)(d[3] * a.group + r % a.group) * HD;
#pragma unroll
  for (int i = 0; i < V; ++i)
    out[i * 32 + lane] = L > 0.0f ? o[i] / L : L == 0.0f ? 0.0f : L;
}
