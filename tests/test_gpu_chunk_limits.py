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


@pytest.mark.parametrize("f16", [False, True])
def test_pages_beyond_32_bits(gpu_lib, f16):
    """Pages whose bytes lie beyond 2^32 in their pool, and rows of q and out
    whose floats lie beyond 2^31: as pages and rows at the beginning.  The
    same of l3g_kv_copy_pages, which brings them there."""
    import torch
    rng = np.random.default_rng(3)
    n, kv, hd = 5, 700, 128
    cache = Paged(rng, [(kv, 0)], 1, hd, f16, spare=0)
    q = rng.normal(0, 1.3, (n, 4, hd)).astype(np.float32)
    run = Run(gpu_lib, cache, [n], 4, q)
    run()
    want = run.got()[0]
    small = run.pools[0]
    page_bytes = small[0].numel() * small.element_size()
    pages = (1 << 32) // page_bytes + 1000
    big = torch.empty(pages, *small.shape[1:], dtype=small.dtype, device="cuda")
    ids = lambda v: torch.tensor([int(i) for i in v], dtype=torch.int32, device="cuda")  # noqa: E731
    have = cache.table[0, 0]
    there = pages - 1 - np.arange(len(have))
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    src, dst = ids(have), ids(there)
    gpu_lib.kv_copy_pages(small.data_ptr(), small.shape[0], big.data_ptr(), pages, page_bytes // ops_ref.PAGE,
                          src.data_ptr(), dst.data_ptr(), 0, len(have), status.data_ptr())
    torch.cuda.synchronize()
    assert not status.any()
    run.table.copy_(torch.from_numpy(there.astype(np.int32).reshape(cache.table.shape)))
    run.desc[0]["pool"], run.desc[0]["n_pages"] = big.data_ptr(), pages
    run.upload()
    run.out.fill_(float("nan"))
    run()
    assert np.array_equal(run.got()[0], want) and run.op.status() == (0, 0)
    # rows 2^29 floats apart
    ld = 1 << 29
    far = torch.empty(4 * ld + 1024, device="cuda")
    for i in range(n):
        far[i * ld:i * ld + 512] = torch.from_numpy(q[i].reshape(-1)).cuda()
    run.op.run(run.seqs.data_ptr(), 1, n, far.data_ptr(), ld, far.data_ptr() + 2048, ld)
    torch.cuda.synchronize()
    for i in range(n):
        assert np.array_equal(far[i * ld + 512:i * ld + 1024].cpu().numpy().reshape(4, hd), want[i])
    assert run.op.status() == (0, 0)


@pytest.mark.parametrize("mag", [1e36, 1e-36])
@pytest.mark.parametrize("unseen", [False, True])
def test_values_near_the_ends_of_the_range(gpu_lib, mag, unseen):
    """V so large that the weights' own scale (2^13) would take a finite mean
    beyond fp32, and as small; also where a row's tile is taken again for an
    unseen NaN."""
    rng = np.random.default_rng(10)
    n, kv = 9, 100
    cache = Paged(rng, [(kv, 0)], 1, 64, False)
    q = rng.normal(0, 1.3, (n, 4, 64)).astype(np.float32)
    cache.v[0] *= np.float32(mag)
    for p in cache.pools:
        p[:, :, 1] *= np.float32(mag)
    run = Run(gpu_lib, cache, [n], 4, q)
    if unseen:
        run.pools[0][cache.table[0, 0, 0], kv - 1, 1, 3] = float("nan")
    run()
    got = run.got()[0]
    want = ops_ref.attention(q, (cache.k[0], cache.v[0]), n, kv)
    bound = ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))
    assert np.abs(got[:-1] - want[:-1]).max() <= bound
    last = np.abs(got[-1] - want[-1])
    assert np.isnan(last[:, 3]).all() if unseen else last.max() <= bound
    assert np.delete(last, 3, 1).max() <= bound
    assert run.op.status() == (0, 0)
