"""Log probabilities of rows of several slices (l3g_logprobs_*): whole slices
of the type's lowest value, of other large negative values, of infinities and
of NaN, against 64 bits."""
import numpy as np
import pytest

import ops_ref

pytestmark = pytest.mark.gpu

SLICE = 8192


def _run(gpu_lib, x, targets, k):
    import torch
    n, v = x.shape
    xd, td = torch.from_numpy(x).cuda(), torch.from_numpy(np.asarray(targets, np.int32)).cuda()
    f = dict(device="cuda", dtype=torch.float32)
    i = dict(device="cuda", dtype=torch.int32)
    o = {"lp": torch.empty(n, **f), "ent": torch.empty(n, **f), "rank": torch.empty(n, **i),
         "ids": torch.empty(n, k, **i), "tlp": torch.empty(n, k, **f)}
    op = gpu_lib.LogProbs(n, v)
    op.run(xd.data_ptr(), v, n, td.data_ptr(), *(o[a].data_ptr() for a in ("lp", "ent", "rank")), k,
           o["ids"].data_ptr(), o["tlp"].data_ptr())
    assert op.status() == (0, 0)
    return {a: b.cpu().numpy() for a, b in o.items()}


@pytest.mark.parametrize("v", [20000, 128256, 128257])
@pytest.mark.parametrize("low", [float(np.finfo(np.float32).min), -1e38, -1e35, -1e30, -np.inf])
def test_masked_slices(gpu_lib, v, low):
    rng = np.random.default_rng(v)
    x = rng.normal(0, 2, (6, v)).astype(np.float32)
    x[0, SLICE:] = low                       # all but the first slice
    x[1, :SLICE] = low                       # the first
    x[2, :] = low                            # everywhere but in one place
    x[2, v - 1] = 0.5
    x[3, SLICE // 2:v - SLICE // 2] = low    # slices in the middle and parts of two
    x[4, :] = low                            # everywhere
    x[5, rng.random(v) < 0.7] = low          # here and there
    t = [5, SLICE + 3, v - 1, v - 2, 9, 1234]
    o = _run(gpu_lib, x, t, 5)
    for r in range(6):
        lp, ent, rank, ids, tlp = ops_ref.logprobs(x[r], t[r], 5)
        if r == 4 and low == -np.inf:
            assert o["lp"][r] == -np.inf and o["ent"][r] == 0 and (o["tlp"][r] == -np.inf).all()
        else:
            # log S, x - m and S's terms in fp32: 2^-19, and 2^-22 of the spread (20) of what counts
            if np.isfinite(lp):
                assert abs(o["lp"][r] - lp) <= 2.0 ** -19 + 2.0 ** -22 * max(20.0, abs(lp)), (r, o["lp"][r], lp)
            else:
                assert o["lp"][r] == lp
            assert abs(o["ent"][r] - ent) <= 2.0 ** -19 + 2.0 ** -22 * 80, (r, o["ent"][r], ent)
            np.testing.assert_allclose(o["tlp"][r], tlp, rtol=2.0 ** -21, atol=2.0 ** -17)
        assert o["rank"][r] == rank and np.array_equal(o["ids"][r], ids)


def test_infinite_and_nan_slices(gpu_lib):
    v = 128256
    rng = np.random.default_rng(1)
    x = rng.normal(0, 2, (4, v)).astype(np.float32)
    x[0, 3 * SLICE:5 * SLICE] = np.nan
    x[1, 2 * SLICE:3 * SLICE] = np.inf
    x[2, :] = np.finfo(np.float32).min
    x[2, 100000] = np.nan
    x[3, :] = np.nan
    o = _run(gpu_lib, x, [7, 2 * SLICE + 4, 0, 3], 3)
    for r in range(4):
        assert np.isnan(o["lp"][r]) and np.isnan(o["ent"][r]) and np.isnan(o["tlp"][r]).all(), r
    assert o["rank"][1] == 4 and np.array_equal(o["ids"][1], 2 * SLICE + np.arange(3))


@pytest.mark.parametrize("v,k", [(170001, 64), (300000, 40), (600001, 64)])
def test_many_slices(gpu_lib, v, k):
    """More keys of the slices than are compared with each other (1024), and
    than shared memory holds (2048): places by search in the slices' lists."""
    rng = np.random.default_rng(v)
    x = rng.normal(0, 3, (5, v)).astype(np.float32)
    x[1] = rng.integers(0, 4, v)             # ties over every slice
    x[2] = np.arange(v)                      # all alternatives in the last slice
    x[3] = -np.arange(v)                     # in the first
    x[4] = -np.inf
    x[4, ::9000] = 1.0                       # fewer than k beside the masked
    t = [7, v - 1, v - 2, 3, 9000]
    o = _run(gpu_lib, x, t, k)
    for r in range(5):
        lp, ent, rank, ids, tlp = ops_ref.logprobs(x[r], t[r], k)
        # (a row of 600000 distinct whole numbers: what counts spreads over 20)
        assert abs(o["lp"][r] - lp) <= 2.0 ** -19 + 2.0 ** -22 * max(20.0, abs(lp)), (r, o["lp"][r], lp)
        assert abs(o["ent"][r] - ent) <= 2.0 ** -19 + 2.0 ** -22 * 80, (r, o["ent"][r], ent)
        assert o["rank"][r] == rank and np.array_equal(o["ids"][r], ids), r
        np.testing.assert_allclose(o["tlp"][r], tlp, rtol=2.0 ** -21, atol=2.0 ** -17)


def test_rows_beyond_32_bits(gpu_lib):
    """Logits of more than 2^31 bytes times 2: the last rows as the first."""
    import torch
    v, n = 128256, 8400  # 4.3 GB
    x = torch.randn(n, v, device="cuda") * 2
    t = torch.arange(n, dtype=torch.int32, device="cuda") * 3
    lp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    ids = torch.empty(n, 3, dtype=torch.int32, device="cuda")
    op = gpu_lib.LogProbs(n, v)
    op.run(x.data_ptr(), v, n, t.data_ptr(), lp.data_ptr(), ent.data_ptr(), 0, 3, ids.data_ptr())
    assert op.status() == (0, 0)
    for r in (0, 4186, 8373, 8374, 8399):
        row = x[r].cpu().numpy()
        a, b, _, c, _ = ops_ref.logprobs(row, 3 * r, 3)
        assert abs(lp[r].item() - a) <= 2.0 ** -19 + 2.0 ** -22 * 40
        assert abs(ent[r].item() - b) <= 2.0 ** -19 + 2.0 ** -22 * 80
        assert np.array_equal(ids[r].cpu().numpy(), c)
