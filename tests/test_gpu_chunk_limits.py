"""Chunk attention (l3g_chunk_attn_run) at the ends of its ranges: as many
sequences as a call takes, and magnitudes that differ within a tile of the
cache."""
import math

import numpy as np
import pytest

import ops_ref
from ops_ref import Paged
from test_gpu_chunk_attention import Run

pytestmark = pytest.mark.gpu

SEQS_MAX = 512  # L3G_CHUNK_SEQS_MAX


@pytest.mark.parametrize("f16", [False, True])
def test_sequences_of_a_call(gpu_lib, f16):
    rng = np.random.default_rng(1)
    lens = [(int(n), int(max(n, k))) for n, k in zip(rng.integers(0, 4, SEQS_MAX), rng.integers(1, 40, SEQS_MAX))]
    lens[-1] = (3, 300)
    cache = Paged(rng, [(k, 0) for _, k in lens], 1, 32, f16)
    chunks = [n for n, _ in lens]
    q = rng.normal(0, 1.3, (sum(chunks), 2, 32)).astype(np.float32)
    run = Run(gpu_lib, cache, chunks, 2, q)
    run()
    got, at = run.got(), 0
    for i, (n, k) in enumerate(lens):
        if n:
            want = ops_ref.attention(q[at:at + n], (cache.k[i], cache.v[i]), n, k)
            bound = ops_ref.attention_bound(q[at:at + n], (cache.k[i], cache.v[i]))
            assert np.abs(got[i] - want).max() <= bound, i
        at += n
    assert run.op.status() == (0, 0)
    p = run.q.data_ptr()
    for n in (SEQS_MAX + 1, -1):
        with pytest.raises(gpu_lib.L3GError, match="n_seqs=%d" % n):
            run.op.run(run.seqs.data_ptr(), n, run.rows, p, run.ldq, run.out.data_ptr(), run.ldo)


@pytest.mark.parametrize("which", [0, 1])
def test_magnitudes_differ_in_a_tile(gpu_lib, which):
    """An f32 cache whose channels (V) or positions (K) differ by up to 2^22.
    An operand keeps 22 bits of each value down to 2^-17 of its tile's
    largest, and below that an absolute 2^-39 of it (half the lo term's last
    place): so each output channel to its own magnitude's bound plus that."""
    rng = np.random.default_rng(2)
    n, kv, hd = 30, 500, 64
    cache = Paged(rng, [(kv, 0)], 1, hd, False)
    q = rng.normal(0, 1.3, (n, 4, hd)).astype(np.float32)
    if which:
        f = np.ldexp(np.float32(1), -(np.arange(hd) % 23)).astype(np.float32)
        cache.v[0] *= f
        for p in cache.pools:
            p[:, :, 1] *= f
    else:
        f = np.ldexp(np.float32(1), -(np.arange(kv) % 23)).astype(np.float32)
        cache.k[0] *= f[:, None]
        for j in range(-(-kv // ops_ref.PAGE)):
            m = min(ops_ref.PAGE, kv - j * ops_ref.PAGE)
            cache.pools[0][cache.table[0, 0, j], :m, 0] *= f[j * ops_ref.PAGE:j * ops_ref.PAGE + m, None]
    run = Run(gpu_lib, cache, [n], 4, q)
    run()
    got = run.got()[0]
    want = ops_ref.attention(q, (cache.k[0], cache.v[0]), n, kv)
    # scores: as ops_ref.attention_bound, with each channel's own largest V
    S = np.linalg.norm(q.astype(np.float64), axis=-1).max() * \
        np.linalg.norm(cache.k[0].astype(np.float64), axis=-1).max() / math.sqrt(hd)
    V = np.abs(cache.v[0].astype(np.float64)).max(axis=(0, 1))
    bound = V * (2 * S * 2.0 ** -20 + 2.0 ** -20) + V.max() * 2.0 ** -38
    err = np.abs(got - want).max(axis=(0, 1))
    assert (err <= bound).all(), (err / bound).max()
    assert run.op.status() == (0, 0)
