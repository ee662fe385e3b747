// Log probabilities of given tokens, entropy, rank and top alternatives of
// logits rows (included by l3g_ops.cu inside namespace l3g).
#pragma once

struct LogprobArgs {
  const float* x;
  long long ld;
  int n, vocab, k;
  const int* targets;
  float* logprob;
  float* entropy;
  int* rank;
  int* top_ids;
  float* top_lp;
};

// The order of the alternatives: larger logit first, lower id on ties (-0
// and +0 tie).
__device__ __forceinline__ uint64_t logit_key(float v, int idx) {
  return topk_key(v == 0.0f ? 0.0f : v, idx);
}

// One CTA of 256 threads per row: maximum, sums, rank, then one pass per
// alternative.
__global__ void k_logprobs_simple(const LogprobArgs a) {
  __shared__ float red[8], red2[8];
  __shared__ int redi[8];
  __shared__ uint64_t redk[8];
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* x = a.x + (long long)r * a.ld;
  float m = -INFINITY;
  for (int i = tid; i < a.vocab; i += 256) m = fmaxf(m, x[i]);
  m = warp_max(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  __syncthreads();
  const int t = a.targets ? a.targets[r] : -1;
  const bool has_t = t >= 0 && t < a.vocab;
  const float xt = has_t ? x[t] : 0.0f;
  const uint64_t kt = has_t ? logit_key(xt, t) : ~0ull;
  float s = 0.0f, s1 = 0.0f;
  int before = 0;
  for (int i = tid; i < a.vocab; i += 256) {
    const float v = x[i], d = v - m;
    if (v != -INFINITY) {
      const float e = expf(d);
      s += e;
      s1 = fmaf(e, d, s1);
    }
    before += logit_key(v, i) > kt;
  }
  s = warp_sum(s);
  s1 = warp_sum(s1);
  for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) {
    red[warp] = s;
    red2[warp] = s1;
    redi[warp] = before;
  }
  __syncthreads();
  s = 0.0f, s1 = 0.0f, before = 0;
  for (int w = 0; w < 8; ++w) {
    s += red[w];
    s1 += red2[w];
    before += redi[w];
  }
  const bool none = m == -INFINITY && s == 0.0f;
  const float ls = logf(s);
  if (tid == 0) {
    if (a.logprob) a.logprob[r] = !has_t ? __int_as_float(0x7fc00000) : none ? -INFINITY : xt - m - ls;
    if (a.rank) a.rank[r] = has_t ? before : -1;
    if (a.entropy) a.entropy[r] = none ? 0.0f : ls - s1 / s;
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = 0;
    for (int i = tid; i < a.vocab; i += 256) {
      const uint64_t key = logit_key(x[i], i);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) redk[warp] = best;
    __syncthreads();
    for (int w = 0; w < 8; ++w) best = max(best, redk[w]);
    last = best;
    if (tid == 0) {
      if (a.top_ids) a.top_ids[(size_t)r * a.k + j] = key_index(best);
      if (a.top_lp) a.top_lp[(size_t)r * a.k + j] = none ? -INFINITY : key_value(best) - m - ls;
    }
  }
}
