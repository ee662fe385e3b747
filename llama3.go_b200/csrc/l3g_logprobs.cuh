// Log probabilities of given tokens, entropy, rank and top alternatives of
// logits rows (included by l3g_ops.cu inside namespace l3g).
//
// With m = max x, d_i = x_i - m, S = sum e^d_i, S1 = sum e^d_i d_i:
//   log p_t = d_t - log S,   entropy = log S - S1 / S,
// so one pass over the row is enough and nothing cancels (d_i <= 0).  A row is
// cut into slices that a CTA holds in registers; slices with maxima m_a are
// joined by S = sum_a S_a e^(m_a - m), S1 = sum_a (S1_a + S_a (m_a - m)) e^(m_a - m).
// 4 bytes and about 26 instructions a value, with alternatives; 512 x 128256 with 20
// of them take 107 us, 2.46 TB/s: neither memory (34% under ncu) nor the issue slots
// (54%) are full, the slices' chains of barriers and the threshold's search bound it.
#pragma once

constexpr int LP_THREADS = 256;
// Values of a slice: 32 a thread.  With 16, rows have twice the slices to join:
// 1 to 24 rows x 128256 with 20 alternatives take 30 to 42 us instead of 19 to
// 24, 512 rows 188 instead of 107, 131 x 8000 11.8 instead of 9.6.
constexpr int LP_E = 32, LP_SLICE = LP_THREADS * LP_E;
constexpr int LP_CAND = 1024;  // gathered keys
// Threads with a key at or above the threshold that the search stops at: k and
// up to LP_SLACK more.
constexpr int LP_SLACK = 16;

struct LogprobArgs {
  const float* x;
  long long ld;
  int n, vocab, k, slices;
  const int* targets;
  float* logprob;
  float* entropy;
  int* rank;
  int* top_ids;
  float* top_lp;
  Result* res;
  unsigned long long wait_ns;
  float4* part;     // [n][slices] {m, S, S1, tokens before the target (bits)}
  uint64_t* part_k; // [n][slices][k] the slices' top keys, sorted
};

// The order of the alternatives: larger logit first, lower id on ties (-0
// and +0 tie).
__device__ __forceinline__ uint64_t logit_key(float v, int idx) {
  return topk_key(v == 0.0f ? 0.0f : v, idx);
}

// What a row's sums give.
struct LogprobRow {
  float m, s, s1;
  int before;
};
__device__ __forceinline__ void logprob_write(const LogprobArgs& a, int r, const LogprobRow& w,
                                              float xt, bool has_t, int tid) {
  const bool none = w.m == -INFINITY && w.s == 0.0f;  // every token masked
  if (tid != 0) return;
  const float ls = logf(w.s);
  if (a.logprob)
    a.logprob[r] = !has_t ? __int_as_float(0x7fc00000) : none ? -INFINITY : xt - w.m - ls;
  if (a.rank) a.rank[r] = has_t ? w.before : -1;
  if (a.entropy) a.entropy[r] = none ? 0.0f : ls - w.s1 / w.s;
}
__device__ __forceinline__ void logprob_top(const LogprobArgs& a, int r, const LogprobRow& w,
                                            uint64_t key, int place) {
  const bool none = w.m == -INFINITY && w.s == 0.0f;
  if (a.top_ids) a.top_ids[(size_t)r * a.k + place] = key_index(key);
  if (a.top_lp)
    a.top_lp[(size_t)r * a.k + place] = none ? -INFINITY : key_value(key) - w.m - logf(w.s);
}

// Slices of LP_SLICE values, dealt to as many CTAs as fit at once.  VEC:
// rows start on 16-byte boundaries; a slice then comes by one bulk copy into
// shared memory while the slice before is worked on, so that memory is never
// idle: a slice's chain of barriers (maximum, sums and threshold, candidates)
// takes longer than its bytes need.  Few threads with many values each: what a
// thread does once per slice costs as much as its values.
//
// The top k of the slice: the k-th largest of the threads' own largest values
// is at or below the slice's k-th value, so every one of the top k belongs to a
// thread whose largest is at or above it.  One warp bisects that threshold, on
// the values' bits, until k to k + LP_SLACK threads are at or above it; their
// values at or above it are gathered as keys (value and id) and each finds its
// place by counting the larger ones.  The work hardly depends on the values: a
// descending row costs what a random one does.  Where too many threads tie, too
// many values are at or above the threshold, or the slice holds a NaN or +inf,
// the k keys are found one by one.
constexpr int LP_SMEM = 2 * LP_SLICE * 4;
template <bool VEC>
__global__ void __launch_bounds__(LP_THREADS, 3) k_logprobs_part(const LogprobArgs a) {
  constexpr int NWARP = LP_THREADS / 32;
  constexpr int E = LP_E, SLICE = LP_SLICE;
  __shared__ uint64_t full[2];
  __shared__ int abort_flag;
  __shared__ float red[NWARP], red2[NWARP], redm[NWARP], best_of[LP_THREADS];
  __shared__ int redi[NWARP], count;
  __shared__ uint32_t low32, slow;
  __shared__ uint64_t cand[LP_CAND];
  L3G_DYNAMIC_SMEM(lp_buf);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  const unsigned total = (unsigned)a.n * a.slices;  // (max_rows x slices is below 2^31)
  // thread 0: the copy of the CTA's i-th slice
  auto fetch = [&](int i) {
    const unsigned at = blockIdx.x + i * gridDim.x;
    if (at >= total) return;
    const unsigned row = at / a.slices;
    const int base = (int)(at - row * a.slices) * SLICE;
    const int cnt = a.vocab - base < SLICE ? a.vocab - base : SLICE;
    const uint32_t bytes = (uint32_t)(cnt & ~3) * 4;  // the last values are read as they are
    mbar_arrive_expect_tx(&full[i & 1], bytes);
    if (bytes)
      bulk_g2s(lp_buf + (size_t)(i & 1) * SLICE * 4, a.x + (long long)row * a.ld + base, bytes,
               &full[i & 1]);
  };
  if (VEC && tid == 0) {
    mbar_init(&full[0], 1);
    mbar_init(&full[1], 1);
    abort_flag = 0;
    fence_mbar_init();
    fetch(0);
  }
  // the row's target and its logit, a slice ahead
  auto target = [&](unsigned at) {
    return a.targets && at < total ? a.targets[at / a.slices] : -1;
  };
  auto logit = [&](unsigned at, int t) {
    return t >= 0 && t < a.vocab ? a.x[(long long)(at / a.slices) * a.ld + t] : 0.0f;
  };
  int t = target(blockIdx.x);
  float xt = logit(blockIdx.x, t);
  int round = 0;
  for (unsigned at = blockIdx.x; at < total; at += gridDim.x, ++round) {
    const int r = (int)(at / a.slices), slice = (int)(at - (unsigned)r * a.slices);
    const int base = slice * SLICE;
    const float* x = a.x + (long long)r * a.ld;
    const bool has_t = t >= 0 && t < a.vocab;
    const int t_next = target(at + gridDim.x);
    // value e of thread tid: id base + (e / 4 * LP_THREADS + tid) * 4 + e % 4
    auto id_of = [&](int e) { return base + (e / 4 * LP_THREADS + tid) * 4 + e % 4; };
    __syncthreads();  // the slice before is done with shared memory
    if (tid == 0) count = 0;
    if (VEC) {
      if (tid == 0) fetch(round + 1);
      if (!mbar_wait(&full[round & 1], round >> 1 & 1, &abort_flag, a.res, 60, a.wait_ns))
        abort_flag = 1;
    }
    const float* buf = reinterpret_cast<const float*>(lp_buf) + (size_t)(round & 1) * SLICE;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const int id = id_of(e);
      if (VEC && id + 3 < a.vocab) {
        const float4 f = *reinterpret_cast<const float4*>(buf + id - base);
        v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e + i] = id + i < a.vocab ? x[id + i] : -INFINITY;
      }
    }
    // this thread's largest value (NaNs left out)
    float tm = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; e += 2) tm = fmaxf(fmaxf(tm, v[e]), v[e + 1]);
    best_of[tid] = tm;
    const float wm = warp_max(tm);
    if (lane == 0) redm[warp] = wm;
    __syncthreads();
    if (VEC && *(volatile int*)&abort_flag) return;  // (uniform: set before the barrier)
    const float m = warp_max(redm[lane % NWARP]);
    // a slice of nothing but -inf (and NaN) is taken relative to 0
    const float mm = m == -INFINITY ? 0.0f : m;
    unsigned long long s2 = 0ull, t2 = 0ull;  // pairs: sums of p, of p d
    const unsigned long long nm2 = pk2(-mm, -mm), l2e = pk2(1.44269504f, 1.44269504f);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const unsigned long long d2 = add2(pk2(v[e], v[e + 1]), nm2);
      const float2 u = upk2(mul2(d2, l2e)), d = upk2(d2);
      const unsigned long long p2 = pk2(ex2(u.x), ex2(u.y));
      s2 = add2(s2, p2);
      // (p is 0 from d = -127 on; -inf times that would be NaN)
      t2 = fma2(p2, pk2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), t2);
    }
    // tokens before the target: ids below it from xt on, ids above it beyond xt
    // (values past the vocabulary are -inf, with ids beyond the target's)
    int before = 0;
    if (has_t && tm >= xt) {  // (few threads hold a value beyond a likely token's)
      if (base > t) {
#pragma unroll
        for (int e = 0; e < E; ++e) before += v[e] > xt;
      } else if (base + SLICE <= t) {
#pragma unroll
        for (int e = 0; e < E; ++e) before += v[e] >= xt;
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) before += v[e] > xt || (v[e] == xt && id_of(e) < t);
      }
    }
    const float2 sp = upk2(s2), tp = upk2(t2);
    const float s = warp_sum(sp.x + sp.y), s1 = warp_sum(tp.x + tp.y);
    before = (int)__reduce_add_sync(0xffffffffu, (unsigned)before);
    if (lane == 0) {
      red[warp] = s;
      red2[warp] = s1;
      redi[warp] = before;
    }
    const float xt_next = logit(at + gridDim.x, t_next);
    __syncthreads();
    LogprobRow w{m, 0.0f, 0.0f, 0};
    const bool last = a.slices == 1;
    if (warp == 0 || last) {
#pragma unroll
      for (int i = 0; i < NWARP; ++i) {
        w.s += red[i];
        w.s1 += red2[i];
        w.before += redi[i];
      }
    }
    if (last)
      logprob_write(a, r, w, xt, has_t, tid);
    else if (tid == 0)
      a.part[(size_t)r * a.slices + slice] = make_float4(w.m, w.s, w.s1, __int_as_float(w.before));
    t = t_next;
    xt = xt_next;
    if (a.k == 0) continue;

    // the threshold as an ordered integer: count(tm >= lo) >= k, count(tm >= hi) < k
    auto key32 = [](float f) {
      const uint32_t b = __float_as_uint(f == 0.0f ? 0.0f : f);
      return b & 0x80000000u ? ~b : b | 0x80000000u;
    };
    if (warp == 0) {
      uint32_t b[NWARP];
#pragma unroll
      for (int i = 0; i < NWARP; ++i) b[i] = key32(best_of[i * 32 + lane]);
      auto at_least = [&](uint32_t k32) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < NWARP; ++i) c += b[i] >= k32;
        return (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
      };
      // steps down from the largest, doubling, then halves
      uint32_t lo = 0, hi = key32(m) + 1, step = 1u << 20;
      int c = 0, at_lo = LP_THREADS;  // threads at or above lo
      while (lo == 0 && hi > step) {
        const uint32_t mid = hi - step;
        step <<= 1;
        c = at_least(mid);
        if (c >= a.k) lo = mid, at_lo = c;
        else hi = mid;
      }
      while (hi - lo > 1 && at_lo > a.k + LP_SLACK) {
        const uint32_t mid = lo + (hi - lo) / 2;
        c = at_least(mid);
        if (c >= a.k) lo = mid, at_lo = c;
        else hi = mid;
      }
      if (lane == 0) {
        low32 = lo;
        slow = at_lo > a.k + LP_SLACK || !(w.s < INFINITY);
      }
    }
    __syncthreads();
    if (!slow && key32(tm) >= low32) {
      // the places of its values at or above the threshold, then those one by one
      const float thr = __uint_as_float(low32 & 0x80000000u ? low32 & 0x7fffffffu : ~low32);
      uint32_t set = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) set |= (v[e] < thr ? 0u : 1u) << e;
      while (set) {
        const int e = __ffs(set) - 1;
        set &= set - 1;
        const int id = id_of(e);
        if (id < a.vocab) {
          // (read again: no registers by index)
          const uint64_t key = logit_key(VEC && (id | 3) < a.vocab ? buf[id - base] : x[id], id);
          const int place = atomicAdd(&count, 1);
          if (place < LP_CAND) cand[place] = key;
        }
      }
    }
    __syncthreads();
    int n = count;
    if (slow || n > LP_CAND) {  // one by one: the largest key below the last
      n = 0;
      uint64_t below = ~0ull;
      bool first = true;
      for (; n < a.k; ++n) {
        uint64_t best = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint64_t key = id_of(e) < a.vocab ? logit_key(v[e], id_of(e)) : 0ull;
          if ((key < below || first) && key > best) best = key;
        }
        __syncthreads();  // cand[n] is not yet in use, or was cleared by all
        if (tid == 0) cand[n] = 0ull;
        __syncthreads();
        atomicMax(reinterpret_cast<unsigned long long*>(&cand[n]), (unsigned long long)best);
        __syncthreads();
        below = cand[n];
        first = false;
        if (below == 0ull) break;  // no values left
      }
    }
    for (int i = tid; i < n; i += LP_THREADS) {
      const uint64_t key = cand[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) place += cand[j] > key;
      if (place < a.k) {
        if (last)
          logprob_top(a, r, w, key, place);
        else
          a.part_k[((size_t)r * a.slices + slice) * a.k + place] = key;
      }
    }
    if (!last)  // a slice of fewer than k values
      for (int i = n + tid; i < a.k; i += LP_THREADS)
        a.part_k[((size_t)r * a.slices + slice) * a.k + i] = 0ull;
  }
}

// Joins a row's slices; a key's place is the number of larger ones in the
// slices' sorted lists: of all keys where there are few, else by searching the
// lists, in shared memory where they fit.  grid rows.
constexpr int LP_JOIN = 256, LP_LISTS = 2048, LP_PAIRS = 1024;
static __global__ void __launch_bounds__(LP_JOIN) k_logprobs_join(const LogprobArgs a) {
  __shared__ uint64_t keys[LP_LISTS];
  __shared__ float4 sums;
  const int r = blockIdx.x, tid = threadIdx.x;
  const int t = a.targets ? a.targets[r] : -1;
  const bool has_t = t >= 0 && t < a.vocab;
  const float xt = has_t ? a.x[(long long)r * a.ld + t] : 0.0f;
  const int n = a.slices * a.k;
  pdl_wait();
  const float4* part = a.part + (size_t)r * a.slices;
  const uint64_t* lists = a.part_k + (size_t)r * n;
  if (tid < 32) {  // a lane the slices lane, lane + 32 ..; then a tree over lanes
    float m = -INFINITY;
    for (int i = tid; i < a.slices; i += 32) m = fmaxf(m, part[i].x);
    m = warp_max(m);
    float s = 0.0f, s1 = 0.0f;
    int before = 0;
    for (int i = tid; i < a.slices; i += 32) {
      const float4 p = part[i];
      // a slice of nothing but -inf: its sums are 0 (NaN, if it has one)
      const float d = p.x == -INFINITY ? 0.0f : p.x - m;
      const float f = p.x == -INFINITY ? 1.0f : ex2(d * 1.44269504f);
      s = fmaf(p.y, f, s);
      // (f is 0 from d = -150 on; S d of a slice of a mask's lowest values is
      // beyond fp32's range, and -inf times that 0 would be NaN)
      s1 = fmaf(fmaf(p.y, fmaxf(d, -1e30f), p.z), f, s1);
      before += __float_as_int(p.w);
    }
    s = warp_sum(s);
    s1 = warp_sum(s1);
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (tid == 0) sums = make_float4(m, s, s1, __int_as_float(before));
  }
  const bool fit = n <= LP_LISTS;
  if (fit)
    for (int i = tid; i < n; i += LP_JOIN) keys[i] = lists[i];
  __syncthreads();
  const LogprobRow w{sums.x, sums.y, sums.z, __float_as_int(sums.w)};
  logprob_write(a, r, w, xt, has_t, tid);
  if (n <= LP_PAIRS) {  // few keys: against every other one
    for (int i = tid; i < n; i += LP_JOIN) {
      const uint64_t key = keys[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) place += keys[j] > key;
      if (key != 0ull && place < a.k) logprob_top(a, r, w, key, place);
    }
    return;
  }
  const uint64_t* from = fit ? keys : lists;
  for (int i = tid; i < n; i += LP_JOIN) {
    const uint64_t key = from[i];
    if (key == 0ull) continue;
    const int own = i / a.k;
    int place = i % a.k;
    for (int j = 0; j < a.slices && place < a.k; ++j) {
      if (j == own) continue;
      const uint64_t* l = from + (size_t)j * a.k;
      int lo = 0, hi = a.k;  // keys of the list above this one
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (l[mid] > key) lo = mid + 1;
        else hi = mid;
      }
      place += lo;
    }
    if (place < a.k) logprob_top(a, r, w, key, place);
  }
}
