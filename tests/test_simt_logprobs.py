"""The log probability and page copy kernels on the CPU, under the SIMT
emulator: bulk copies and their barriers, slices and their join, the search of
the alternatives, strides and alignment, and values at the ends of the type."""
import numpy as np
import pytest

import ops_ref
import simt_ops_lib

LOWEST = float(np.finfo(np.float32).min)
SLICE = 8192  # values that a CTA takes at once


def _close(got, want, spread):
    """log S, x - m and S's terms in fp32: 2^-19 absolute and 2^-22 of the
    spread of the values that count."""
    assert abs(float(got) - float(want)) <= 2.0 ** -19 + 2.0 ** -22 * spread, (got, want)


def _check_row(o, r, x, t, k, spread):
    lp, ent, rank, ids, tlp = ops_ref.logprobs(x, t, k)
    if np.isfinite(lp):
        _close(o["lp"][r], lp, max(spread, abs(lp)))
    _close(o["ent"][r], ent, 4 * spread)
    assert o["rank"][r] == rank
    if k:
        assert np.array_equal(o["ids"][r], ids)
        with np.errstate(over="ignore"):
            np.testing.assert_allclose(o["tlp"][r], tlp.astype(np.float32), rtol=2.0 ** -21, atol=2.0 ** -17)


@pytest.mark.parametrize("n,v,k,ld,shift,seed", [
    (2, 97, 20, 100, 0, 3), (1, 1, 1, None, 0, None), (2, 8193, 5, None, 0, 4), (2, 20000, 64, None, 0, None),
    (1, 8191, 3, None, 1, 5), (2, 16390, 8, 16392, 0, 6), (3, 300, 0, 301, 0, 7)])
def test_rows(n, v, k, ld, shift, seed):
    rng = np.random.default_rng(v + k)
    x = rng.normal(0, 3, (n, v)).astype(np.float32)
    t = rng.integers(0, v, n)
    o = simt_ops_lib.logprobs(x, t, k, ld=ld, shift=shift, seed=seed)
    for r in range(n):
        _check_row(o, r, x[r], t[r], k, float(x[r].max() - x[r].min()))


@pytest.mark.parametrize("low", [LOWEST, -1e38, -1e35, -1e30])
def test_slices_of_the_lowest_values(low):
    """Whole slices of a mask's large negative values: they count for nothing,
    and neither the entropy nor anything else is NaN.  (A slice's sum is taken
    relative to its own maximum, so S = 8192 and S (m_slice - m) is beyond
    fp32's range.)"""
    v = 2 * SLICE + 100
    rng = np.random.default_rng(2)
    x = rng.normal(0, 2, (4, v)).astype(np.float32)
    x[0, SLICE:] = low                       # a slice and a part of one
    x[1, :SLICE] = low                       # the first
    x[2, :] = low                            # everywhere but in one place
    x[2, SLICE + 7] = 0.5
    x[3, :] = low                            # everywhere
    t = [5, SLICE + 3, SLICE + 7, 9]
    o = simt_ops_lib.logprobs(x, t, 3)
    for r in range(4):
        lp, ent, rank, ids, _ = ops_ref.logprobs(x[r], t[r], 3)
        _close(o["lp"][r], lp, 20.0)
        _close(o["ent"][r], ent, 80.0)
        assert o["rank"][r] == rank and np.array_equal(o["ids"][r], ids)


def test_slices_of_infinities_and_nan():
    v = 2 * SLICE + 100
    rng = np.random.default_rng(3)
    x = rng.normal(0, 2, (4, v)).astype(np.float32)
    x[0, :SLICE] = -np.inf
    x[1, SLICE:] = np.nan
    x[2, SLICE:] = np.inf
    x[3, :] = LOWEST
    x[3, SLICE + 5] = np.nan
    o = simt_ops_lib.logprobs(x, [SLICE + 1, 4, SLICE + 2, 1], 2)
    _check_row(o, 0, x[0], SLICE + 1, 2, 20.0)
    for r in (1, 2, 3):
        assert np.isnan(o["lp"][r]) and np.isnan(o["ent"][r]) and np.isnan(o["tlp"][r]).all(), r
    assert np.array_equal(o["ids"][2], [SLICE, SLICE + 1]) and o["rank"][2] == 2


def test_ties_over_slices():
    v, k = 2 * SLICE, 40
    rng = np.random.default_rng(4)
    x = np.stack([np.zeros(v), rng.integers(0, 3, v)]).astype(np.float32)
    x[0, ::2] = -0.0
    o = simt_ops_lib.logprobs(x, [SLICE, 77], k)
    for r, t in enumerate((SLICE, 77)):
        _check_row(o, r, x[r], t, k, 2.0)


def test_copy_pages():
    rng = np.random.default_rng(5)
    pool = rng.integers(0, 256, (9, ops_ref.PAGE, 48), dtype=np.uint8)
    src, dst, rows = [0, 3, 7, 2], [1, 8, 5, 4], [256, 37, 0, 1]
    want = pool.copy()
    for a, b, n in zip(src, dst, rows):
        want[b, :n] = pool[a, :n]
    got, status = simt_ops_lib.copy_pages(pool, None, src, dst, rows)
    assert status == (0, 0) and np.array_equal(got, want)
    other = rng.integers(0, 256, (3, ops_ref.PAGE, 48), dtype=np.uint8)
    want = other.copy()
    want[2] = pool[8]
    # whole pages; entries outside their bounds are skipped and noted
    got, status = simt_ops_lib.copy_pages(pool, other, [8, 9], [2, 0])
    assert status == (4, 1) and np.array_equal(got, want)
    for s, d, r in (([-1], [0], [1]), ([0], [3], [1]), ([0], [-1], [1]), ([0], [0], [257]), ([0], [0], [-1])):
        got, status = simt_ops_lib.copy_pages(pool, other, s, d, r)
        assert status == (4, 0) and np.array_equal(got, other)
    # more entries than grid rows
    want = other.copy()
    want[0, :5], want[1, :6], want[2, :7] = pool[3, :5], pool[4, :6], pool[5, :7]
    got, _ = simt_ops_lib.copy_pages(pool, other, [3, 4, 5], [0, 1, 2], [5, 6, 7], max_rows=2)
    assert np.array_equal(got, want)
