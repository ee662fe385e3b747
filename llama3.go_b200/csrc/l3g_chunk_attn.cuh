// Attention of ragged chunks of new tokens over paged caches (included by
// l3g_ops.cu inside namespace l3g).
#pragma once

struct ChunkArgs {
  const l3g_chunk_seq* seqs;
  int n_seqs, total_q;
  const float* q;
  long long ldq;
  float* out;
  long long ldo;
  int layer, heads, hkv, group;
  float scale;
  Result* res;
};

// Whether a descriptor stays inside its bounds (its pages are checked where
// they are read).
__device__ __forceinline__ bool chunk_seq_ok(const l3g_chunk_seq& s, int total_q) {
  return s.pool && s.pages && s.pps >= 0 && s.q0 >= 0 && s.n_q >= 0 && s.n_q <= total_q &&
         s.q0 <= total_q - s.n_q && s.kv_len >= 0 &&
         (long long)s.kv_len <= (long long)s.pps * KV_PAGE;
}

// One warp per (token, query head): the online softmax over the positions the
// token sees, lane = dims lane + 32 j.  grid (blocks of 8 warps, sequences).
template <int HD, typename KT>
__global__ void k_chunk_simple(const ChunkArgs a) {
  constexpr int DPL = HD / 32;
  const int lane = threadIdx.x & 31;
  const l3g_chunk_seq s = a.seqs[blockIdx.y];
  if (!chunk_seq_ok(s, a.total_q)) {
    if (threadIdx.x == 0 && blockIdx.x == 0) report(a.res, ERR_SEQ, blockIdx.y);
    return;
  }
  for (int w = blockIdx.x * 8 + (threadIdx.x >> 5); w < s.n_q * a.heads; w += gridDim.x * 8) {
    const int t = w / a.heads, h = w % a.heads, kvh = h / a.group;
    const float* q = a.q + (long long)(s.q0 + t) * a.ldq + (size_t)h * HD;
    float qv[DPL], o[DPL], m = -INFINITY, l = 0.0f;
    for (int j = 0; j < DPL; ++j) {
      qv[j] = q[lane + 32 * j];
      o[j] = 0.0f;
    }
    const int* pages = s.pages + ((size_t)a.layer * a.hkv + kvh) * s.pps;
    const int see = s.kv_len - s.n_q + t + 1;
    bool bad = false;
    for (int p = 0; p < see; ++p) {
      const int page = pages[p / KV_PAGE];
      if (page < 0 || page >= s.n_pages) {
        if (lane == 0) report(a.res, ERR_PAGE, page);
        bad = true;
        break;
      }
      const KT* row = reinterpret_cast<const KT*>(s.pool) +
                      ((size_t)page * KV_PAGE + (p & (KV_PAGE - 1))) * 2 * HD;
      float d = 0.0f;
      for (int j = 0; j < DPL; ++j) d = fmaf(qv[j], (float)row[lane + 32 * j], d);
      const float sc = warp_sum(d) * a.scale;
      const float mn = fmaxf(m, sc);
      const float c = m == -INFINITY ? 0.0f : expf(m - mn), e = expf(sc - mn);
      l = fmaf(l, c, e);
      for (int j = 0; j < DPL; ++j) o[j] = fmaf(o[j], c, e * (float)row[HD + lane + 32 * j]);
      m = mn;
    }
    if (bad) continue;
    float* out = a.out + (long long)(s.q0 + t) * a.ldo + (size_t)h * HD;
    for (int j = 0; j < DPL; ++j) out[lane + 32 * j] = see > 0 ? o[j] / l : 0.0f;
  }
}
