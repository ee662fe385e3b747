"""The serving operators in 64 bits (numpy), from their definitions, and the
paged caches that their tests run on."""
import math

import numpy as np

PAGE = 256


class Paged:
    """Pools of pages and the page tables of sequences over them: seqs is a
    list of (kv_len, pool index).  Rows that no sequence holds are NaN."""

    def __init__(self, rng, seqs, hkv, hd, f16, layers=1, pools=1, spare=2, pps_extra=0):
        self.hkv, self.hd, self.layers = hkv, hd, layers
        self.dt = np.float16 if f16 else np.float32
        self.lens = [k for k, _ in seqs]
        self.pps = max(1, max(-(-k // PAGE) for k in self.lens)) + pps_extra
        need = [0] * pools
        for k, p in seqs:
            need[p] += layers * hkv * -(-k // PAGE)
        self.pool_of = [p for _, p in seqs]
        self.pools = [np.full((n + spare, PAGE, 2, hd), np.nan, self.dt) for n in need]
        free = [list(rng.permutation(n + spare)) for n in need]
        self.table = np.zeros((len(seqs), layers * hkv, self.pps), np.int32)
        self.k, self.v = [], []
        for s, (n, p) in enumerate(seqs):
            kk = rng.normal(0, 1, (layers * hkv, n, hd)).astype(self.dt)
            vv = rng.normal(0, 1, (layers * hkv, n, hd)).astype(self.dt)
            self.k.append(kk)
            self.v.append(vv)
            for h in range(layers * hkv):
                for j in range(-(-n // PAGE)):
                    page = free[p].pop()
                    self.table[s, h, j] = page
                    m = min(PAGE, n - j * PAGE)
                    self.pools[p][page, :m, 0] = kk[h, j * PAGE:j * PAGE + m]
                    self.pools[p][page, :m, 1] = vv[h, j * PAGE:j * PAGE + m]


def attention(q, cells, n_q, kv_len, scale=None):
    """q [n_q][H][hd], cells = (K, V) [hkv][kv_len][hd] -> [n_q][H][hd] in
    float64; tokens that see nothing are zero."""
    K, V = (c.astype(np.float64) for c in cells)
    H, hd = q.shape[1:]
    G = H // K.shape[0]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out = np.zeros(q.shape, np.float64)
    for t in range(n_q):
        see = kv_len - n_q + t + 1
        if see <= 0:
            continue
        for h in range(H):
            s = K[h // G, :see] @ q[t, h].astype(np.float64) * scale
            w = np.exp(s - s.max())
            out[t, h] = (w / w.sum()) @ V[h // G, :see]
    return out


def attention_bound(q, cells, scale=None):
    """Elementwise error bound of an fp32 implementation whose operands carry
    at least 22 bits: a score is off by at most (2^-22 + 2^-22) of
    scale |q||k| for the operands' rounding and 2^-21 for a sum of up to 128
    products in 32 bits with truncation (16 steps of 2^-23 and half of it
    for the fp32 exponent argument), so by S 2^-20; weights then by the
    factor exp(S 2^-20), the weighted mean by twice that times the largest
    |v|, plus 2^-20 |v| for the second product and the normalization."""
    K, V = cells
    hd = q.shape[-1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    if not K.size or not q.size:
        return 0.0
    S = scale * np.linalg.norm(q.astype(np.float64), axis=-1).max() * \
        np.linalg.norm(K.astype(np.float64), axis=-1).max()
    return float(np.abs(V.astype(np.float64)).max() * (2 * S * 2.0 ** -20 + 2.0 ** -20))


def logprobs(x, target, k):
    """One row: (logprob, entropy, rank, ids, logprobs) in float64."""
    x = np.asarray(x, np.float64)
    v = np.where(x == 0, 0.0, x)
    order = np.lexsort((np.arange(x.size), -v))
    m = x.max()
    if m == -np.inf:
        lp = np.full(x.size, -np.inf)
        ent = 0.0
    else:
        e = np.exp(x - m)
        lp = x - m - np.log(e.sum())
        p = e / e.sum()
        ent = -(p[p > 0] * lp[p > 0]).sum()
    t_ok = 0 <= target < x.size
    rank = int(np.nonzero(order == target)[0][0]) if t_ok else -1
    return (lp[target] if t_ok else np.nan), ent, rank, order[:k], lp[order[:k]]
