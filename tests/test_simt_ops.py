"""The serving operators' kernels on the CPU, under the SIMT emulator: the
arithmetic, the split of the cache axis over CTAs, the barriers under random
schedules, and descriptors and pages outside their bounds."""
import numpy as np
import pytest

import ops_ref
import simt_ops_lib
from ops_ref import Paged


def _queries(rng, n, heads, hd):
    return rng.normal(0, 1.3, (n, heads, hd)).astype(np.float32)


def _check(cache, chunks, heads, q, out, skip=()):
    at = 0
    for i, n in enumerate(chunks):
        qi, got = q[at:at + n], out[at:at + n].reshape(n, heads, cache.hd)
        at += n
        if i in skip or n == 0:
            continue
        cells = (cache.k[i], cache.v[i])
        want = ops_ref.attention(qi, cells, n, cache.lens[i])
        assert np.isfinite(got).all(), i
        assert np.abs(got - want).max() <= ops_ref.attention_bound(qi, cells), (i, np.abs(got - want).max())
    assert np.isnan(out[at:]).all()


@pytest.mark.parametrize("heads,hkv,hd,f16,lens,grid,seed", [
    (4, 2, 64, True, [(1, 70), (3, 3), (40, 300)], 3, None),
    (4, 2, 64, True, [(1, 70), (3, 3), (40, 300)], 5, 11),
    (4, 2, 64, False, [(1, 70), (3, 3), (40, 300)], 4, 12),
    (3, 1, 32, True, [(50, 260), (0, 9), (2, 0), (5, 3)], 2, 13),
    (3, 1, 32, False, [(50, 260), (1, 64), (2, 65)], 7, 14),
    (8, 1, 128, True, [(17, 500), (1, 129)], 2, 15),
    (2, 1, 128, False, [(1, 700), (65, 130)], 6, 16),
])
def test_chunk_attention(heads, hkv, hd, f16, lens, grid, seed):
    rng = np.random.default_rng(heads * 3 + hd)
    cache = Paged(rng, [(k, 0) for _, k in lens], hkv, hd, f16)
    chunks = [n for n, _ in lens]
    q = _queries(rng, sum(chunks), heads, hd)
    out, err, where = simt_ops_lib.chunk_attention(cache, chunks, heads, q, grid=grid, seed=seed)
    assert (err, where) == (0, 0)
    _check(cache, chunks, heads, q, out)


def test_chunk_attention_descriptors_outside_their_bounds():
    rng = np.random.default_rng(5)
    lens = [(4, 100), (6, 90), (3, 300)]
    chunks = [n for n, _ in lens]
    cache = Paged(rng, [(k, 0) for _, k in lens], 1, 32, True)
    q = _queries(rng, 13, 2, 32)
    for field, value in (("n_q", -1), ("q0", 1 << 30), ("kv_len", 100000), ("kv_len", -5), ("q0", -2),
                         ("n_q", 1 << 30), ("pool", 0), ("pages", 0)):
        def edit(desc):
            desc[1][field] = value
        out, err, where = simt_ops_lib.chunk_attention(cache, chunks, 2, q, edit=edit)
        assert (err, where) == (3, 1), field
        _check(cache, chunks, 2, q, out, skip=(1,))
        assert np.isnan(out[4:10]).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page", [-1, 1 << 20])
def test_chunk_attention_bad_page(f16, page):
    rng = np.random.default_rng(6)
    lens = [(4, 100), (6, 90), (3, 600)]
    chunks = [n for n, _ in lens]
    cache = Paged(rng, [(k, 0) for _, k in lens], 2, 32, f16)
    q = _queries(rng, 13, 4, 32)
    table = cache.table.copy()
    table[2, 1, 1] = page
    for grid in (1, 4):  # whole row tiles, and pieces that are joined
        out, err, where = simt_ops_lib.chunk_attention(cache, chunks, 4, q, table=table, grid=grid)
        assert (err, where) == (4, page)
        _check(cache, chunks, 4, q, np.where(np.arange(15)[:, None] < 10, out, np.nan), skip=(2,))
        assert np.isnan(out[10:13].reshape(3, 4, 32)[:, 2:]).all()


@pytest.mark.parametrize("f16", [False, True])
def test_chunk_attention_unseen_nan(f16):
    """A NaN in V reaches the tokens that see it and no other."""
    rng = np.random.default_rng(7)
    n, kv, p = 20, 150, 140
    cache = Paged(rng, [(kv, 0)], 1, 32, f16)
    q = _queries(rng, n, 2, 32)
    pools = [x.copy() for x in cache.pools]
    pools[0][cache.table[0, 0, 0], p, 1, 3] = np.nan
    out, err, _ = simt_ops_lib.chunk_attention(cache, [n], 2, q, pools=pools)
    got = out[:n].reshape(n, 2, 32)
    cells = (cache.k[0], cache.v[0])
    want = ops_ref.attention(q, cells, n, kv)
    first = p - (kv - n)
    assert err == 0 and np.abs(got[:first] - want[:first]).max() <= ops_ref.attention_bound(q, cells)
    assert np.isnan(got[first:, :, 3]).all()
    rest = np.delete(got[first:], 3, 2) - np.delete(want[first:], 3, 2)
    assert np.abs(rest).max() <= ops_ref.attention_bound(q, cells)
