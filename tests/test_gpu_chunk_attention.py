"""Attention of ragged token chunks over paged caches (l3g_chunk_attn_*)
against the definition in 64 bits, through the C ABI: cache types, head
layouts, chunk lengths from none to several row tiles, caches that end inside
a page or a tile, tokens that see nothing, row strides, several pools and
layers, NaN and infinities in places that a token does not see, descriptors
and pages outside their bounds, streams and captured graphs."""
import math

import numpy as np
import pytest

import ops_ref
from ops_ref import PAGE, Paged

pytestmark = pytest.mark.gpu


class Run:
    """One call's device side: pools, tables, q, out (NaN-filled)."""

    def __init__(self, gpu_lib, cache, chunks, heads, q, q0s=None, ldq=None, ldo=None, extra_rows=3):
        import torch
        self.torch, self.l3g, self.cache, self.chunks = torch, gpu_lib, cache, chunks
        self.heads, self.hd = heads, cache.hd
        width = heads * cache.hd
        self.total = sum(chunks)
        self.rows = (max(q0s[i] + n for i, n in enumerate(chunks)) if q0s else self.total) + extra_rows
        self.ldq, self.ldo = ldq or width, ldo or width
        self.q0 = list(q0s) if q0s else list(np.concatenate([[0], np.cumsum(chunks)[:-1]]).astype(int))
        qh = np.full((self.rows, self.ldq), np.nan, np.float32)
        at = 0
        for i, n in enumerate(chunks):
            qh[self.q0[i]:self.q0[i] + n, :width] = q[at:at + n].reshape(n, width)
            at += n
        self.q = torch.from_numpy(qh).cuda()
        self.out = torch.full((self.rows, self.ldo), float("nan"), device="cuda")
        self.pools = [torch.from_numpy(p).cuda() for p in cache.pools]
        self.table = torch.from_numpy(cache.table).cuda()
        self.desc = gpu_lib.chunk_seqs(len(chunks))
        for i, n in enumerate(chunks):
            p = self.pools[cache.pool_of[i]]
            d = self.desc[i]
            d["pool"], d["n_pages"] = p.data_ptr(), p.shape[0]
            d["pages"] = self.table.data_ptr() + i * cache.layers * cache.hkv * cache.pps * 4
            d["pps"], d["q0"], d["n_q"], d["kv_len"] = cache.pps, self.q0[i], n, cache.lens[i]
        self.seqs = torch.from_numpy(self.desc.view(np.uint8)).cuda()
        self.op = gpu_lib.ChunkAttention(heads, cache.hkv, cache.hd,
                                         gpu_lib.L3G_KV_F16 if cache.dt == np.float16 else gpu_lib.L3G_KV_F32)

    def upload(self):
        self.seqs.copy_(self.torch.from_numpy(self.desc.view(np.uint8)))

    def __call__(self, layer=0, scale=0.0, stream=0):
        self.op.run(self.seqs.data_ptr(), len(self.chunks), self.rows, self.q.data_ptr(), self.ldq,
                    self.out.data_ptr(), self.ldo, layer, scale, stream)

    def got(self):
        self.torch.cuda.synchronize()
        o = self.out.cpu().numpy()
        return [o[self.q0[i]:self.q0[i] + n, :self.heads * self.hd].reshape(n, self.heads, self.hd)
                for i, n in enumerate(self.chunks)]


def _queries(rng, n, heads, hd):
    return rng.normal(0, 1.3, (n, heads, hd)).astype(np.float32)


def _check(run, cache, q, layer=0, scale=None):
    got, at = run.got(), 0
    hk = cache.hkv
    for i, n in enumerate(run.chunks):
        cells = (cache.k[i][layer * hk:(layer + 1) * hk], cache.v[i][layer * hk:(layer + 1) * hk])
        qi = q[at:at + n]
        at += n
        if n == 0:
            continue
        want = ops_ref.attention(qi, cells, n, cache.lens[i], scale)
        assert np.isfinite(got[i]).all(), i
        err = np.abs(got[i] - want)
        assert err.max() <= ops_ref.attention_bound(qi, cells, scale), (i, err.max())
        norm = np.linalg.norm(want)
        # single errors are independent: their norm stays far below the bound
        assert np.linalg.norm(got[i] - want) <= 4e-6 * norm + 1e-30, (i, np.linalg.norm(got[i] - want) / norm)
    assert run.op.status() == (0, 0)


# heads, kv heads, head_dim
SHAPES = [(32, 8, 128), (4, 2, 64), (6, 2, 32), (24, 8, 128), (8, 1, 64), (7, 1, 128), (5, 5, 32), (2, 1, 128)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,hkv,hd", SHAPES)
def test_ragged_chunks(gpu_lib, heads, hkv, hd, f16):
    rng = np.random.default_rng(heads * 131 + hkv * 17 + hd + f16)
    # single tokens, chunks at position 0, lengths around a tile, a page and a row tile's tokens
    lens = [(1, 1), (1, 300), (3, 3), (17, 129), (33, 256), (40, 257), (1, 700), (130, 600), (0, 50), (5, 127)]
    if heads * hd >= 3000:
        lens = lens[:8]
    cache = Paged(rng, [(k, 0) for _, k in lens], hkv, hd, f16)
    q = _queries(rng, sum(n for n, _ in lens), heads, hd)
    run = Run(gpu_lib, cache, [n for n, _ in lens], heads, q)
    run()
    _check(run, cache, q)
    # rows behind the last sequence stay as they were
    assert np.isnan(run.out[run.total:].cpu().numpy()).all()


@pytest.mark.parametrize("f16", [False, True])
def test_long_cache_few_rows(gpu_lib, f16):
    """A few tokens over long caches: the cache axis is split and joined."""
    rng = np.random.default_rng(7)
    lens = [(1, 5000), (2, 4097), (1, 33), (4, 2000)]
    cache = Paged(rng, [(k, 0) for _, k in lens], 2, 128, f16)
    q = _queries(rng, 8, 8, 128)
    run = Run(gpu_lib, cache, [n for n, _ in lens], 8, q)
    run()
    _check(run, cache, q)
    first = run.out.clone()
    for _ in range(3):  # the same bits from every call
        run()
        assert run.torch.equal(run.out.nan_to_num(), first.nan_to_num())


@pytest.mark.parametrize("f16", [False, True])
def test_tokens_that_see_nothing(gpu_lib, f16):
    rng = np.random.default_rng(8)
    lens = [(4, 0), (200, 130), (1, 0), (3, 3), (64, 1)]
    cache = Paged(rng, [(k, 0) for _, k in lens], 2, 64, f16)
    q = _queries(rng, sum(n for n, _ in lens), 8, 64)
    run = Run(gpu_lib, cache, [n for n, _ in lens], 8, q)
    run()
    _check(run, cache, q)
    got = run.got()
    assert not got[0].any() and not got[1][:70].any() and not got[2].any() and not got[4][:63].any()


def test_strides_orders_layers_pools(gpu_lib):
    rng = np.random.default_rng(9)
    lens = [(5, 70), (1, 260), (9, 9), (130, 400)]
    cache = Paged(rng, [(lens[0][1], 0), (lens[1][1], 1), (lens[2][1], 0), (lens[3][1], 1)], 2, 64, True, layers=3,
                  pools=2, pps_extra=3)
    q = _queries(rng, sum(n for n, _ in lens), 4, 64)
    # the sequences' rows in another order, with rows between them that belong to none
    run = Run(gpu_lib, cache, [n for n, _ in lens], 4, q, q0s=[150, 141, 0, 10], ldq=4 * 64 + 12, ldo=4 * 64 + 4)
    for layer, scale in ((0, None), (2, 0.3)):
        run.out.fill_(float("nan"))
        run(layer=layer, scale=scale or 0.0)
        _check(run, cache, q, layer, scale)
        out = run.out.cpu().numpy()
        assert np.isnan(out[:, 256:]).all() and np.isnan(out[9]).all() and np.isnan(out[155:]).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_unseen_values_do_not_matter(gpu_lib, f16, bad):
    """A NaN or an infinity at position p reaches the tokens from p on (as
    NaN) and no earlier one."""
    rng = np.random.default_rng(10)
    n, kv, p = 70, 330, 290
    cache = Paged(rng, [(kv, 0)], 1, 64, f16)
    q = _queries(rng, n, 4, 64)
    for which in (0, 1):
        run = Run(gpu_lib, cache, [n], 4, q)
        page = cache.table[0, 0, p // PAGE]
        run.pools[0][page, p % PAGE, which, 5] = bad
        run()
        got = run.got()[0]
        first = p - (kv - n)
        cells = (cache.k[0], cache.v[0])
        want = ops_ref.attention(q, cells, n, kv)
        assert np.abs(got[:first] - want[:first]).max() <= ops_ref.attention_bound(q, cells)
        if which == 1:  # only the dimension that holds it
            assert not np.isfinite(got[first:, :, 5]).any()
            rest = np.delete(got[first:], 5, axis=2) - np.delete(want[first:], 5, axis=2)
            assert np.abs(rest).max() <= ops_ref.attention_bound(q, cells)
        elif math.isnan(bad):
            assert np.isnan(got[first:]).all()
        assert run.op.status() == (0, 0)


@pytest.mark.parametrize("mag", [1e-6, 1.0, 1e4])
def test_magnitudes_f32(gpu_lib, mag):
    """Values far from one, in q, K and V, keep their relative precision."""
    rng = np.random.default_rng(11)
    cache = Paged(rng, [(200, 0)], 1, 64, False)
    for a in (cache.k[0], cache.v[0]):
        a *= np.float32(mag)
    for p in cache.pools:
        p *= np.float32(mag)
    q = _queries(rng, 20, 4, 64) / np.float32(mag)
    run = Run(gpu_lib, cache, [20], 4, q)
    run()
    _check(run, cache, q)


def test_large_scores(gpu_lib):
    """Scores of hundreds: the softmax is taken from its maximum on."""
    rng = np.random.default_rng(12)
    cache = Paged(rng, [(500, 0)], 1, 128, True)
    q = _queries(rng, 33, 4, 128)
    run = Run(gpu_lib, cache, [33], 4, q)
    run(scale=4.0)
    got = run.got()[0]
    cells = (cache.k[0], cache.v[0])
    want = ops_ref.attention(q, cells, 33, 500, 4.0)
    assert np.abs(got - want).max() <= ops_ref.attention_bound(q, cells, 4.0)


def test_descriptors_outside_their_bounds(gpu_lib):
    """Bad descriptors and page ids are skipped and reported; the others run."""
    rng = np.random.default_rng(13)
    lens = [(4, 300), (6, 100), (3, 520)]
    for field, value in (("n_q", -1), ("q0", 1 << 30), ("kv_len", 100000), ("kv_len", -5), ("q0", -2),
                         ("n_q", 1 << 30), ("pool", 0), ("pages", 0)):
        cache = Paged(rng, [(k, 0) for _, k in lens], 2, 64, True)
        q = _queries(rng, 13, 4, 64)
        run = Run(gpu_lib, cache, [n for n, _ in lens], 4, q)
        run.desc[1][field] = value
        run.upload()
        run()
        got = run.got()
        assert run.op.status() == (3, 1), field
        assert run.op.status() == (0, 0)
        for i, a in ((0, 0), (2, 10)):
            want = ops_ref.attention(q[a:a + lens[i][0]], (cache.k[i], cache.v[i]), *lens[i])
            assert np.abs(got[i] - want).max() < 1e-3, (field, i)
        assert np.isnan(got[1]).all(), field
    for page in (-1, 1 << 20):
        cache = Paged(rng, [(k, 0) for _, k in lens], 2, 64, True)
        q = _queries(rng, 13, 4, 64)
        run = Run(gpu_lib, cache, [n for n, _ in lens], 4, q)
        run.table[2, 1, 1] = page
        run()
        got = run.got()
        assert run.op.status() == (4, page)
        for i, a in ((0, 0), (1, 4)):
            want = ops_ref.attention(q[a:a + lens[i][0]], (cache.k[i], cache.v[i]), *lens[i])
            assert np.abs(got[i] - want).max() < 1e-3
        assert np.isnan(got[2][:, 2:]).all()  # the heads of the bad page's kv head
        run.table[2, 1, 1] = int(cache.table[2, 1, 1])  # and the handle works again
        run()
        _check(run, cache, q)


def test_streams_and_graph_replay(gpu_lib):
    """On another stream, and captured: a replay follows the descriptors that
    are in memory then."""
    import torch
    rng = np.random.default_rng(14)
    lens = [(2, 900), (40, 300)]
    cache = Paged(rng, [(k, 0) for _, k in lens], 2, 64, True)
    q = _queries(rng, 42, 8, 64)
    run = Run(gpu_lib, cache, [n for n, _ in lens], 8, q)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    run(stream=st.cuda_stream)
    _check(run, cache, q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(stream=torch.cuda.current_stream().cuda_stream)
    run.out.fill_(float("nan"))
    g.replay()
    _check(run, cache, q)
    cache.lens = [600, 77]  # shorter caches of the same pages
    for i, k in enumerate(cache.lens):
        run.desc[i]["kv_len"] = k
        cache.k[i], cache.v[i] = cache.k[i][:, :k], cache.v[i][:, :k]
    run.upload()
    g.replay()
    _check(run, cache, q)


def test_refusals(gpu_lib):
    import torch
    op = gpu_lib.ChunkAttention(4, 2, 64, gpu_lib.L3G_KV_F32)
    b = torch.zeros(4096, device="cuda")
    p = b.data_ptr()
    op.run(0, 0, 0, 0, 256, 0, 256)  # nothing to do
    for args, msg in (((p, -1, 1, p, 256, p, 256), "n_seqs"), ((p, 1025, 1, p, 256, p, 256), "n_seqs"),
                      ((p, 1, -1, p, 256, p, 256), "total_q"), ((0, 1, 1, p, 256, p, 256), "null"),
                      ((p, 1, 1, p, 255, p, 256), "strides"), ((p, 1, 1, p, 256, p, 258), "strides"),
                      ((p, 1, 1, p + 4, 256, p, 256), "aligned"), ((p, 1, 1, p, 256, p, 256, -1), "layer"),
                      ((p, 1, 1, p, 256, p, 256, 0, float("nan")), "scale")):
        with pytest.raises(gpu_lib.L3GError, match=msg):
            op.run(*args)
    op.Close()
    with pytest.raises(gpu_lib.L3GError, match="null"):
        op.run(p, 1, 1, p, 256, p, 256)
