"""Infinities in K under the SIMT emulator: an infinite score as the formula
has it, a weight of zero where it is negative and NaN where it is positive, in
the tokens that see the key and in no other."""
import numpy as np
import pytest

import ops_ref
import simt_ops_lib
from ops_ref import PAGE, Paged


def _want(q, cells, n, kv):
    with np.errstate(invalid="ignore"):
        w = ops_ref.attention(q, cells, n, kv)
    return w


@pytest.mark.parametrize("hd,heads,hkv,grids", [(32, 2, 1, (1, 3)), (64, 4, 2, (3,)), (128, 6, 1, (2,))])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_infinite_key(hd, heads, hkv, grids, f16, bad):
    rng = np.random.default_rng(hd + heads)
    n, kv = 7, 150
    cache = Paged(rng, [(kv, 0)], hkv, hd, f16)
    q = rng.normal(0, 1.3, (n, heads, hd)).astype(np.float32)
    q[3, 0, 5] = 0.0          # 0 times infinity: NaN
    q[4, 0, 5] = 1e-9         # far below the row's largest: its sign still counts
    q[5, 0, 5] = -1e-9
    bound = ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))
    pools = [x.copy() for x in cache.pools]
    k = cache.k[0].copy()
    for p in (10, 145, 148):  # seen by all, and from tokens 2 and 5 on
        pools[0][cache.table[0, 0, p // PAGE], p % PAGE, 0, 5] = bad
        k[0, p, 5] = bad
    want = _want(q, (k, cache.v[0]), n, kv)
    for grid in grids:
        out, err, _ = simt_ops_lib.chunk_attention(cache, [n], heads, q, pools=pools, grid=grid, seed=grid)
        got = out[:n].reshape(n, heads, hd)
        assert err == 0
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fin = ~np.isnan(want)
        assert fin.any() and not fin.all()
        assert np.abs(got[fin] - want[fin]).max() <= bound


@pytest.mark.parametrize("f16", [False, True])
def test_only_infinite_keys(f16):
    """A token all of whose scores are -inf has no weight left and gets zeros,
    as one that sees no position; an unseen NaN in V changes nothing."""
    rng = np.random.default_rng(8)
    n = kv = 12
    cache = Paged(rng, [(kv, 0)], 1, 32, f16)
    q = np.abs(rng.normal(0, 1.3, (n, 2, 32))).astype(np.float32) + 0.1
    pools = [x.copy() for x in cache.pools]
    k = cache.k[0].copy()
    page = cache.table[0, 0, 0]
    pools[0][page, :3, 0, 4] = -np.inf
    k[0, :3, 4] = -np.inf
    pools[0][page, 11, 1, 7] = np.nan
    out, err, _ = simt_ops_lib.chunk_attention(cache, [n], 2, q, pools=pools)
    got = out[:n].reshape(n, 2, 32)
    assert err == 0 and (got[:3] == 0).all()
    want = ops_ref.attention(q[3:11], (k[:, :11], cache.v[0][:, :11]), 8, 11)
    assert np.abs(got[3:11] - want).max() <= ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))
    assert np.isnan(got[11, :, 7]).all() and np.isfinite(np.delete(got[11], 7, 1)).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_infinite_query(f16, bad):
    """An infinity or a NaN in q gives NaN in its own row and touches no other."""
    rng = np.random.default_rng(9)
    n, kv = 6, 140
    cache = Paged(rng, [(kv, 0)], 1, 32, f16)
    q = rng.normal(0, 1.3, (n, 2, 32)).astype(np.float32)
    q[2, 1, 3] = bad
    out, err, _ = simt_ops_lib.chunk_attention(cache, [n], 2, q)
    got = out[:n].reshape(n, 2, 32)
    q[2, 1, 3] = 0.0
    want = ops_ref.attention(q, (cache.k[0], cache.v[0]), n, kv)
    assert err == 0 and np.isnan(got[2, 1]).all()
    got[2, 1] = want[2, 1]
    assert np.abs(got - want).max() <= ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))


@pytest.mark.parametrize("mag", [1e36, 1e-36])
def test_values_near_the_ends_of_the_range(mag):
    """V so large that the weights' own scale (2^13) would take a finite mean
    beyond fp32, and as small."""
    rng = np.random.default_rng(10)
    n, kv = 5, 70
    cache = Paged(rng, [(kv, 0)], 1, 32, False)
    q = rng.normal(0, 1.3, (n, 2, 32)).astype(np.float32)
    cache.v[0] *= np.float32(mag)
    for p in cache.pools:
        p[:, :, 1] *= np.float32(mag)
    want = ops_ref.attention(q, (cache.k[0], cache.v[0]), n, kv)
    for grid in (1, 2):
        out, err, _ = simt_ops_lib.chunk_attention(cache, [n], 2, q, grid=grid)
        got = out[:n].reshape(n, 2, 32)
        assert err == 0 and np.abs(got - want).max() <= ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))
