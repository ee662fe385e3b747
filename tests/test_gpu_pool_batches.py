"""Batches of states on a shared pool: a call that finds too few pages leaves
the pool, the tables and the caches as they were (l3g_batch_extend,
l3g_batch_step)."""
import numpy as np
import pytest

from conftest import synthetic_model

pytestmark = pytest.mark.gpu


def _load(gpu_lib, name="small"):
    cfg, T = synthetic_model(name)
    m = gpu_lib.LoadModelFromTensors(gpu_lib.hparams_for(cfg), T, gpu_lib.default_options(device=0))
    return cfg, m, cfg.n_layers * cfg.n_heads_kv


def test_a_batch_takes_all_its_pages_or_none(gpu_lib):
    import synthetic
    cfg, m, h = _load(gpu_lib)
    ids = synthetic.prompt_ids(cfg, 400, seed=1)
    batch = gpu_lib.Batch(m, 4)
    pool = m.NewKvPool(3 * h)
    a, b, c = (m.NewStateInPool(pool, 512) for _ in range(3))
    # new pages: two of each (layer, kv head) for each state, three are there
    with pytest.raises(gpu_lib.L3GError, match="KV pool exhausted") as e:
        batch.extend([a, b], [ids[:300], ids[:300]])
    assert e.value.code == gpu_lib.L3G_E_CTX
    assert pool.FreePages == 3 * h and a.Pages == b.Pages == 0 and a.Pos == b.Pos == 0
    batch.extend([a], [ids[:300]])  # one of them finds its pages
    assert a.Pos == 300 and pool.FreePages == h
    # copies: the fork's last page, and a page for c: the first takes one, the
    # second finds none, and what the first took is given back
    f = a.Fork()
    before = [x.read_kv(1, 0, 300) for x in (a, f)]
    with pytest.raises(gpu_lib.L3GError, match="KV pool exhausted"):
        batch.extend([f, c], [ids[300:302], ids[:5]])
    assert pool.FreePages == h and f.Pages == a.Pages == 2 * h and c.Pages == 0
    with pytest.raises(gpu_lib.L3GError, match="KV pool exhausted"):
        batch.step([c, f], [1, 2], [1, 2])
    assert pool.FreePages == h and c.Pages == 0 and [x.Pos for x in (a, f, c)] == [300, 300, 0]
    for x, was in zip((a, f), before):
        for got, want in zip(x.read_kv(1, 0, 300), was):
            assert np.array_equal(got, want)
    # each alone goes on: as states of their own
    batch.extend([f], [ids[300:302]])
    own = m.NewState(512)
    batch.extend([own], [ids[:300]])
    batch.extend([own], [ids[300:302]])
    for got, want in zip(f.read_kv(1, 0, 302), own.read_kv(1, 0, 302)):
        assert np.array_equal(got, want)
    assert pool.FreePages == 0
    for s in (f, a, b, c, own):
        s.Close()
    assert pool.FreePages == 3 * h
    for x in (batch, pool, m):
        x.Close()


def test_two_forks_of_a_batch_share_one_copy(gpu_lib):
    """The last of the states that map a page writes in place."""
    import synthetic
    cfg, m, h = _load(gpu_lib)
    ids = synthetic.prompt_ids(cfg, 310, seed=2)
    batch = gpu_lib.Batch(m, 4)
    pool = m.NewKvPool(3 * h)
    a = m.NewStateInPool(pool, 512)
    batch.extend([a], [ids[:300]])
    f = a.Fork()
    batch.extend([a, f], [ids[300:305], ids[305:310]])  # one page each, one of them new
    assert pool.FreePages == 0 and a.Pos == f.Pos == 305
    for s, chunk in ((a, ids[300:305]), (f, ids[305:310])):
        own = m.NewState(512)
        batch.extend([own], [ids[:300]])
        batch.extend([own], [chunk])
        for layer in range(cfg.n_layers):
            for got, want in zip(s.read_kv(layer, 0, 300), own.read_kv(layer, 0, 300)):
                assert np.array_equal(got, want)
        for got, want in zip(s.read_kv(0, 300, 5), own.read_kv(0, 300, 5)):
            assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)
        own.Close()
    for x in (a, f, batch, pool, m):
        x.Close()


def test_a_fork_holds_only_what_its_source_ingested(gpu_lib):
    """Positions that were mapped, sampled past a stop token or lie behind a
    restored snapshot are none of the session's."""
    import synthetic
    cfg, m, h = _load(gpu_lib)
    ids = synthetic.prompt_ids(cfg, 300, seed=3)
    ws = m.NewWorkspace(512, 40)
    pool = m.NewKvPool(8 * h)
    a = m.NewStateInPool(pool, 512)
    m.Prefill(a, ids[:20], ws)
    m.DecodeSample(a, int(ids[20]), 6, ws, top_k=40, temperature=0.8, seed=5)
    a.Pos = 20
    a.Fork(26).Close()  # back, but they have been ingested
    with pytest.raises(gpu_lib.L3GError, match="fork at position 27"):
        a.Fork(27)
    b = m.NewStateInPool(pool, 512)
    m.Prefill(b, ids[:20], ws)
    m.DecodeSample(b, int(ids[20]), 6, ws, top_k=40, temperature=0.8, seed=5, stop_ids=list(range(cfg.vocab)))
    assert b.Pos < 26
    with pytest.raises(gpu_lib.L3GError, match="fork at position 26"):
        b.Fork(26)
    snap = b.Snapshot()
    m.Prefill(a, ids[20:300], ws)
    a.Restore(snap)
    assert a.Pos == b.Pos
    with pytest.raises(gpu_lib.L3GError, match=f"fork at position {b.Pos + 1}"):
        a.Fork(b.Pos + 1)
    a.Fork(b.Pos).Close()
    for x in (a, b, ws, pool, m):
        x.Close()


def test_states_come_and_go_while_a_pool_is_compacted(gpu_lib):
    """Two threads make, fork, trim and free states of a pool that a third
    compacts: nothing is lost, and the caches hold what they held."""
    import threading

    import synthetic
    cfg, m, h = _load(gpu_lib)
    ids = synthetic.prompt_ids(cfg, 500, seed=4)
    batch = gpu_lib.Batch(m, 4)
    pool = m.NewKvPool(12 * h)
    roots = [m.NewStateInPool(pool, 512) for _ in range(3)]
    for k in range(0, 300, 100):  # pages taken in turn
        batch.extend(roots, [ids[k:k + 100]] * 3)
    gone = m.NewStateInPool(pool, 512)
    batch.extend([gone], [ids[:300]])
    roots[0].Close()
    roots = roots[1:]
    snaps = [s.Snapshot() for s in roots]
    free = pool.FreePages
    errors = []

    def churn(src, n):
        try:
            for i in range(n):
                f = src.Fork(100 + 7 * i)
                g = m.NewStateInPool(pool, 512)
                f2 = f.Fork()
                f.Pos = 50
                f.Trim()
                for s in (f, g, f2):
                    s.Close()
        except Exception as e:  # noqa: BLE001 - reported by the test's thread
            errors.append(e)

    threads = [threading.Thread(target=churn, args=(s, 25)) for s in roots]
    for t in threads:
        t.start()
    rounds = 0
    while any(t.is_alive() for t in threads):
        pool.Compact()
        if rounds == 3:
            gone.Close()
        rounds += 1
    for t in threads:
        t.join()
    assert not errors and rounds > 3
    pool.Compact()
    assert pool.FreePages == free + 2 * h
    for s, snap in zip(roots, snaps):
        assert np.array_equal(s.Snapshot(), snap)
        own = m.NewState(512)
        own.Restore(snap)
        batch.extend([s], [ids[300:305]])
        batch.extend([own], [ids[300:305]])
        for layer in range(cfg.n_layers):
            for got, want in zip(s.read_kv(layer, 0, 305), own.read_kv(layer, 0, 305)):
                assert np.array_equal(got, want)
        own.Close()
    for s in roots + [batch, pool, m]:
        s.Close()
