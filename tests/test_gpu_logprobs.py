"""Log probabilities, entropy, rank and top alternatives (l3g_logprobs_*)
against 64 bits: row counts, vocabularies, strides, ties, masked rows, NaN and
infinities, missing targets and outputs, streams and graphs."""
import math

import numpy as np
import pytest

import ops_ref

pytestmark = pytest.mark.gpu


def _run(gpu_lib, x, targets, k, ld=None, op=None, stream=0, want=("lp", "ent", "rank", "ids", "tlp")):
    import torch
    n, v = x.shape
    ld = ld or v
    buf = np.full((n, ld), np.nan, np.float32)
    buf[:, :v] = x
    xd = torch.from_numpy(buf).cuda()
    td = torch.from_numpy(np.asarray(targets, np.int32)).cuda()
    f = dict(device="cuda", dtype=torch.float32)
    i = dict(device="cuda", dtype=torch.int32)
    o = {"lp": torch.full((n + 1,), 7.0, **f), "ent": torch.full((n + 1,), 7.0, **f),
         "rank": torch.full((n + 1,), 7, **i), "ids": torch.full((n + 1, max(k, 1)), 7, **i),
         "tlp": torch.full((n + 1, max(k, 1)), 7.0, **f)}
    if k:
        o["ids"], o["tlp"] = o["ids"].reshape(-1)[:(n + 1) * k].view(n + 1, k), o["tlp"].view(n + 1, k)
    op = op or gpu_lib.LogProbs(n, v)
    ptr = {a: (o[a].data_ptr() if a in want else 0) for a in o}
    op.run(xd.data_ptr(), ld, n, td.data_ptr(), ptr["lp"], ptr["ent"], ptr["rank"], k, ptr["ids"], ptr["tlp"],
           stream)
    torch.cuda.synchronize()
    o = {a: b.cpu().numpy() for a, b in o.items()}
    for a in o:  # the row behind the last stays as it was
        assert (o[a][n] == 7).all()
        if a not in want:
            assert (o[a] == 7).all()
    return {a: b[:n] for a, b in o.items()}


def _close(got, want, spread):
    """fp32 values: log S and x - m are off by 2^-24 relative each, S's
    terms by the exponential's 2^-22 and its sum by 2^-20 at most (a tree of
    partial sums): a few 2^-20 absolute, plus 2^-22 of the spread x - m."""
    assert abs(got - want) <= 2.0 ** -19 + 2.0 ** -22 * spread, (got, want)


@pytest.mark.parametrize("n,v,k,ld", [(1, 128256, 5, None), (3, 97, 20, 100), (7, 2048, 64, None), (2, 1, 1, None),
                                      (5, 33, 33, 37), (4, 8001, 40, 8003), (150, 500, 3, None),
                                      (2, 130001, 64, 130004), (40, 4097, 0, None), (300, 32000, 8, None)])
def test_rows(gpu_lib, n, v, k, ld):
    rng = np.random.default_rng(n * 7 + v + k)
    x = rng.normal(0, 3, (n, v)).astype(np.float32)
    targets = rng.integers(0, v, n)
    o = _run(gpu_lib, x, targets, k, ld)
    for r in range(0, n, max(1, n // 8)):
        lp, ent, rank, ids, tlp = ops_ref.logprobs(x[r], targets[r], k)
        spread = float(x[r].max() - x[r].min())
        _close(o["lp"][r], lp, spread)
        # the entropy's sum of p (x - m) is off by 2^-20 of the mean |x - m|
        _close(o["ent"][r], ent, 4 * spread)
        assert o["rank"][r] == rank
        if k:
            assert np.array_equal(o["ids"][r], ids)
            for a, b in zip(o["tlp"][r], tlp):
                _close(a, b, spread)


def test_orders_and_ties(gpu_lib):
    """Ascending, descending and equal values, few distinct ones, both zeros:
    the lower id first on ties."""
    v, k = 9000, 64
    rng = np.random.default_rng(3)
    rows = [np.arange(v), -np.arange(v), np.zeros(v), np.where(rng.random(v) < 0.5, -0.0, 0.0),
            rng.integers(0, 3, v), np.repeat(np.arange(9), 1000), np.where(np.arange(v) % 128 == 5, 9.0, 0.0),
            np.where(np.arange(v) >= v - 100, 5.0, rng.normal(0, 1, v))]
    x = np.stack(rows).astype(np.float32)
    targets = [0, v - 1, 4000, 17, 8999, 1, 5, v - 1]
    o = _run(gpu_lib, x, targets, k)
    for r in range(len(rows)):
        lp, ent, rank, ids, tlp = ops_ref.logprobs(x[r], targets[r], k)
        assert np.array_equal(o["ids"][r], ids), r
        assert o["rank"][r] == rank, r
        np.testing.assert_allclose(o["tlp"][r], tlp, rtol=2.0 ** -21, atol=2.0 ** -19)
        np.testing.assert_allclose(o["ent"][r], ent, rtol=2.0 ** -18, atol=2.0 ** -19)


def test_masked_and_odd_rows(gpu_lib):
    v = 5000
    rng = np.random.default_rng(4)
    x = rng.normal(0, 2, (8, v)).astype(np.float32)
    x[0, :] = -np.inf                       # nothing left
    x[1, :] = -np.inf
    x[1, 77] = 3.0                          # one token left
    x[2, rng.random(v) < 0.9] = -np.inf
    x[2, 10] = 1.0
    x[3, 40] = np.nan
    x[4, 41] = np.inf
    x[5, :] = np.finfo(np.float32).min      # the type's lowest value everywhere
    x[6, :] = np.finfo(np.float32).min
    x[6, 4999] = 0.5
    x[7] += 1e4                             # far from zero
    t = [5, 77, 10, 3, 41, 9, 4999, 1234]
    o = _run(gpu_lib, x, t, 6)
    assert o["lp"][0] == -np.inf and o["ent"][0] == 0 and o["rank"][0] == 5
    assert np.array_equal(o["ids"][0], np.arange(6)) and (o["tlp"][0] == -np.inf).all()
    assert o["lp"][1] == 0 and o["ent"][1] == 0 and o["rank"][1] == 0 and o["ids"][1, 0] == 77
    assert o["tlp"][1, 0] == 0 and (o["tlp"][1, 1:] == -np.inf).all()
    for r in (2, 5, 6, 7):
        lp, ent, rank, ids, tlp = ops_ref.logprobs(x[r], t[r], 6)
        # row 7: fp32 spacing at 1e4 is in the inputs already
        _close(o["lp"][r], lp, 16.0)
        _close(o["ent"][r], ent, 64.0)
        assert o["rank"][r] == rank and np.array_equal(o["ids"][r], ids)
        fin = np.isfinite(tlp)
        assert np.array_equal(np.isfinite(o["tlp"][r]), fin)
        np.testing.assert_allclose(o["tlp"][r][fin], tlp[fin], rtol=2.0 ** -21, atol=2.0 ** -17)
    for r in (3, 4):
        assert math.isnan(o["lp"][r]) and math.isnan(o["ent"][r]) and np.isnan(o["tlp"][r]).all()
    assert o["ids"][3, 0] == 40 and o["ids"][4, 0] == 41 and o["rank"][4] == 0


def test_missing_targets_and_outputs(gpu_lib):
    rng = np.random.default_rng(5)
    x = rng.normal(0, 2, (4, 700)).astype(np.float32)
    t = [-1, 700, 3, -2 ** 31]
    o = _run(gpu_lib, x, t, 4)
    assert np.array_equal(np.isnan(o["lp"]), [True, True, False, True])
    assert np.array_equal(o["rank"] < 0, [True, True, False, True])
    base = _run(gpu_lib, x, [1, 2, 3, 4], 4)
    for drop in ("lp", "ent", "rank", "ids", "tlp"):
        want = tuple(a for a in base if a != drop)
        part = _run(gpu_lib, x, [1, 2, 3, 4], 4, want=want)
        for a in want:
            assert np.array_equal(part[a], base[a]), (drop, a)


def test_same_bits_streams_and_graphs(gpu_lib):
    import torch
    rng = np.random.default_rng(6)
    x = rng.normal(0, 2, (9, 60000)).astype(np.float32)
    t = rng.integers(0, 60000, 9)
    op = gpu_lib.LogProbs(16, 60000)
    a = _run(gpu_lib, x, t, 20, op=op)
    st = torch.cuda.Stream()
    b = _run(gpu_lib, x, t, 20, op=op, stream=st.cuda_stream)
    for k in a:
        assert np.array_equal(a[k], b[k])
    xd = torch.from_numpy(x).cuda()
    td = torch.from_numpy(t.astype(np.int32)).cuda()
    lp = torch.zeros(9, device="cuda")
    ids = torch.zeros(9, 20, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.run(xd.data_ptr(), 60000, 9, td.data_ptr(), lp.data_ptr(), 0, 0, 20, ids.data_ptr(), 0,
               torch.cuda.current_stream().cuda_stream)
    y = rng.normal(0, 2, (9, 60000)).astype(np.float32)
    xd.copy_(torch.from_numpy(y))
    g.replay()
    c = _run(gpu_lib, y, t, 20, op=op)
    assert np.array_equal(lp.cpu().numpy(), c["lp"]) and np.array_equal(ids.cpu().numpy(), c["ids"])


def test_refusals(gpu_lib):
    import torch
    op = gpu_lib.LogProbs(4, 100)
    p = torch.zeros(4096, device="cuda").data_ptr()
    op.run(p, 100, 0)  # no rows
    for args, msg in (((p, 100, 5), "n=5"), ((p, 100, -1), "n=-1"), ((p, 99, 1), "row stride"),
                      ((0, 100, 1), "null"), ((p, 100, 1, 0, p), "null"),
                      ((p, 100, 1, p, p, 0, 0, 65, p, p), "top_k"), ((p, 100, 1, p, p, 0, 0, -1, p, p), "top_k"),
                      ((p + 2, 100, 1), "aligned")):
        with pytest.raises(gpu_lib.L3GError, match=msg):
            op.run(*args)
