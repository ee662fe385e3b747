"""Forked, trimmed and compacted states (l3g_state_fork, l3g_state_trim,
l3g_kvpool_compact) and chunks of tokens for many sessions with their log
probabilities (l3g_batch_extend), through the C ABI.

- A fork continues exactly as a state that ingested everything itself, and
  neither sees what the other writes; pages are shared until then.
- Compaction moves pages and changes no result.
- What l3g_batch_extend computes does not depend on where a session's pages
  lie or who else maps them (the same bits), and agrees with l3g_batch_step's
  logits: past layer 0 the int8 activations may round the other way, so the
  bar is the 1e-2 relative L2 of the other batched paths' tests.
"""
import numpy as np
import pytest

import ops_ref
from conftest import synthetic_model

pytestmark = pytest.mark.gpu


def _load(gpu_lib, name, kv=0):
    cfg, T = synthetic_model(name)
    return cfg, gpu_lib.LoadModelFromTensors(gpu_lib.hparams_for(cfg), T,
                                             gpu_lib.default_options(device=0, kv_dtype=kv))


def _heads(cfg):
    return cfg.n_layers * cfg.n_heads_kv


def _logits(m, cfg, s, ws, tokens):
    out = []
    for t in tokens:
        lg = np.empty(cfg.vocab, np.float32)
        m.ForwardIntoWorkspace(s, int(t), lg, ws)
        out.append(lg)
    return np.stack(out)


@pytest.mark.parametrize("name,kv,at", [("small", 0, 300), ("small", 1, 256), ("small-hd128", 1, 255),
                                        ("tiny-g3", 0, 77), ("small", 0, 0)])
def test_forks_continue_on_their_own(gpu_lib, name, kv, at):
    import synthetic
    cfg, m = _load(gpu_lib, name, kv)
    ctx = min(cfg.ctx_len, 512)
    ids = synthetic.prompt_ids(cfg, at + 20, seed=3)
    more = synthetic.prompt_ids(cfg, 10, seed=4)
    ws = m.NewWorkspace(ctx, 40)
    pages = _heads(cfg) * -(-ctx // gpu_lib.KV_PAGE)
    pool = m.NewKvPool(3 * pages)
    a, own_a, own_b = m.NewStateInPool(pool, ctx), m.NewState(ctx), m.NewState(ctx)
    m.Prefill(a, ids[:at + 5], ws)
    b = a.Fork(at)  # five positions back
    used = _heads(cfg) * -(-(at + 5) // gpu_lib.KV_PAGE)
    assert b.Pos == at and a.Pos == at + 5 and pool.FreePages == 3 * pages - used  # nothing copied
    m.Prefill(own_a, ids[:at + 5], ws)
    m.Prefill(own_b, ids[:at], ws)
    # both go on, in turn
    for i in range(5):
        la = _logits(m, cfg, a, ws, ids[at + 5 + i:at + 6 + i])
        lb = _logits(m, cfg, b, ws, more[i:i + 1])
        assert np.array_equal(la, _logits(m, cfg, own_a, ws, ids[at + 5 + i:at + 6 + i])), i
        assert np.array_equal(lb, _logits(m, cfg, own_b, ws, more[i:i + 1])), i
    for layer in range(cfg.n_layers):
        for s, o in ((a, own_a), (b, own_b)):
            for x, y in zip(s.read_kv(layer, 0, s.Pos), o.read_kv(layer, 0, o.Pos)):
                assert np.array_equal(x, y)
    # a fork of a fork outlives both
    c = b.Fork()
    a.Close()
    b.Close()
    assert np.array_equal(_logits(m, cfg, c, ws, more[5:8]), _logits(m, cfg, own_b, ws, more[5:8]))
    # and of a private state: a copy
    d = own_b.Fork(at, ctx)
    own_a.Pos = at
    assert np.array_equal(_logits(m, cfg, d, ws, ids[at:at + 3]), _logits(m, cfg, own_a, ws, ids[at:at + 3]))
    for s in (c, d, own_a, own_b):
        s.Close()
    assert pool.FreePages == 3 * pages
    for x in (ws, pool, m):
        x.Close()


def test_fork_refusals_trim_and_exhaustion(gpu_lib):
    import synthetic
    cfg, m = _load(gpu_lib, "small")
    h = _heads(cfg)
    ids = synthetic.prompt_ids(cfg, 400, seed=5)
    ws = m.NewWorkspace(512, 40)
    pool = m.NewKvPool(2 * h)
    a = m.NewStateInPool(pool, 512)
    m.Prefill(a, ids[:300], ws)
    assert pool.FreePages == 0
    with pytest.raises(gpu_lib.L3GError, match="fork at position 301"):
        a.Fork(301)
    with pytest.raises(gpu_lib.L3GError, match="context length exceeded") as e:
        a.Fork(300, 200)
    assert e.value.code == gpu_lib.L3G_E_CTX
    b = a.Fork()
    before = a.read_kv(1, 0, 300)
    with pytest.raises(gpu_lib.L3GError, match="KV pool exhausted"):  # no page for b's copy
        m.Prefill(b, ids[300:301], ws)
    assert b.Pos == 300 and a.Pos == 300
    b.Pos = 256
    b.Trim()  # shares a's first pages only
    assert b.Pages == h
    with pytest.raises(gpu_lib.L3GError, match="KV pool exhausted"):
        m.Prefill(b, ids[300:301], ws)
    m.Prefill(a, ids[300:303], ws)  # its own pages again: no copy needed
    for x, y in zip(before, a.read_kv(1, 0, 300)):
        assert np.array_equal(x, y)
    a.Pos = 10
    a.Trim()
    assert a.Pages == h and pool.FreePages == h
    m.Prefill(b, ids[300:301], ws)  # now there is one
    assert b.Pos == 257 and pool.FreePages == 0
    own = m.NewState(512)
    m.Prefill(own, np.concatenate([ids[:256], ids[300:301]]), ws)
    for x, y in zip(b.read_kv(1, 0, 257), own.read_kv(1, 0, 257)):
        assert np.array_equal(x, y)
    for s in (a, b, own):
        s.Close()
    assert pool.FreePages == 2 * h
    for x in (ws, pool, m):
        x.Close()


@pytest.mark.parametrize("kv", [0, 1])
def test_compaction_changes_no_result(gpu_lib, kv):
    import synthetic
    cfg, m = _load(gpu_lib, "small", kv)
    h = _heads(cfg)
    ids = synthetic.prompt_ids(cfg, 500, seed=6)
    ws = m.NewWorkspace(512, 40)
    pool = m.NewKvPool(12 * h)
    states = [m.NewStateInPool(pool, 512) for _ in range(4)]
    for k in range(0, 480, 32):  # pages taken in turn
        for i, s in enumerate(states):
            m.Prefill(s, ids[k + i:k + i + 30], ws)
    states.append(states[1].Fork(400))
    states[0].Close()
    states[2].Pos = 100
    states[2].Trim()
    live = states[1:]
    snaps = [s.Snapshot() for s in live]
    free = pool.FreePages
    moved = pool.Compact()
    assert moved > 0 and pool.FreePages == free
    assert pool.Compact() == 0  # in order now
    for s, snap in zip(live, snaps):
        assert np.array_equal(s.Snapshot(), snap)
    for s, snap in zip(live, snaps):  # they go on as before, captured steps too
        own = m.NewState(512)
        own.Restore(snap)
        n = min(3, 512 - s.Pos)
        assert np.array_equal(_logits(m, cfg, s, ws, ids[:n]), _logits(m, cfg, own, ws, ids[:n]))
        own.Close()
    for s in live:
        s.Close()
    assert pool.FreePages == 12 * h
    for x in (ws, pool, m):
        x.Close()


def _score_ref(logits, targets, k):
    cols = [ops_ref.logprobs(x, t, k) for x, t in zip(logits, targets)]
    return [np.array(c) for c in zip(*cols)]


@pytest.mark.parametrize("name,kv", [("small", 0), ("small", 1), ("small-hd128", 1), ("tiny-g3", 0)])
def test_extend_agrees_with_batch_step(gpu_lib, name, kv):
    import synthetic
    cfg, m = _load(gpu_lib, name, kv)
    ctx = min(cfg.ctx_len, 512)
    batch = gpu_lib.Batch(m, 4)
    lens = [(0, 9), (40, 1), (min(ctx - 40, 270), 17)]  # (prefix, chunk)
    ids = [synthetic.prompt_ids(cfg, p + n + 1, seed=20 + i) for i, (p, n) in enumerate(lens)]
    ext = [m.NewState(ctx) for _ in lens]
    step = [m.NewState(ctx) for _ in lens]
    for group in (ext, step):  # the prefixes, alike
        batch.extend(group, [x[:p] for x, (p, _) in zip(ids, lens)])
    for s, t, (p, _) in zip(ext, step, lens):
        assert s.Pos == t.Pos == p
    got = batch.extend(ext, [x[p:p + n] for x, (p, n) in zip(ids, lens)],
                       targets=[x[p + 1:p + n + 1] for x, (p, n) in zip(ids, lens)], top_k=5)
    at = 0
    for i, (p, n) in enumerate(lens):
        logits = []
        for t in ids[i][p:p + n]:
            _, lg = batch.step([step[i]], [int(t)], [1], want_logits=True)
            logits.append(lg[0])
        lp, ent, rank, _, tlp = _score_ref(logits, ids[i][p + 1:p + n + 1], 5)
        sl = slice(at, at + n)
        at += n
        for a, b in ((got["logprob"][sl], lp), (got["entropy"][sl], ent), (got["top_logprobs"][sl], tlp)):
            assert np.linalg.norm(a - b) <= 1e-2 * np.linalg.norm(b), (i, np.linalg.norm(a - b) / np.linalg.norm(b))
        assert ext[i].Pos == step[i].Pos == p + n
        for x, y in zip(ext[i].read_kv(0, 0, p + n), step[i].read_kv(0, 0, p + n)):
            # layer 0: fp32 sums in another order (f16 caches: one rounding of 2^-11)
            tol = 1e-5 if kv == 0 else 2.0 ** -10
            assert np.linalg.norm(x - y) <= tol * np.linalg.norm(y)
    for x in ext + step + [batch, m]:
        x.Close()


def test_sessions_from_one_prefix(gpu_lib):
    """As a server would: a prefix ingested once, forked, the forks extended by
    chunks with their log probabilities, some dropped, the pool compacted, the
    others stepped; against sessions with caches of their own, bit by bit."""
    import synthetic
    cfg, m = _load(gpu_lib, "small")
    h = _heads(cfg)
    ctx = 512
    prefix = synthetic.prompt_ids(cfg, 301, seed=31)
    n = 5
    chunks = [synthetic.prompt_ids(cfg, k, seed=40 + k) for k in (1, 130, 0, 33, 7)]
    pool = m.NewKvPool(2 * h * (n + 1))
    batch, other = gpu_lib.Batch(m, 8), gpu_lib.Batch(m, 8)
    root = m.NewStateInPool(pool, ctx)
    assert batch.extend([root], [prefix]) is None and root.Pos == 301
    forks = [root.Fork() for _ in range(n)]
    assert pool.FreePages == 2 * h * n
    own = []
    for _ in range(n):
        s = m.NewState(ctx)
        other.extend([s], [prefix])
        own.append(s)
    targets = [np.concatenate([c[1:], [-1]]) if len(c) else c for c in chunks]
    a = batch.extend(forks, chunks, targets=targets, top_k=8)
    b = other.extend(own, chunks, targets=targets, top_k=8)
    for k in a:
        assert np.array_equal(a[k], b[k], equal_nan=True), k
    assert [s.Pos for s in forks] == [301 + len(c) for c in chunks]
    last = np.cumsum([len(c) for c in chunks]) - 1
    assert np.isnan(a["logprob"][last[0]]) and a["rank"][last[0]] == -1  # no target
    assert np.isfinite(a["logprob"][last[0] + 1:last[1]]).all()
    # twice the same call on other forks: the same bits
    again = [root.Fork() for _ in range(2)]
    c = batch.extend(again, chunks[3:], targets=targets[3:], top_k=8)
    one = batch.extend([root.Fork()], chunks[3:4], targets=targets[3:4], top_k=8)
    assert np.isfinite(one["entropy"]).all() and np.isfinite(c["entropy"]).all()
    forks[1].Close()
    for s in again:
        s.Close()
    pool.Compact()
    keep = [0, 2, 3, 4]
    ta = tb = [5, 6, 7, 8]
    for _ in range(3):
        ta, la = batch.step([forks[i] for i in keep], ta, [1, 2, 3, 4], want_logits=True)
        tb, lb = other.step([own[i] for i in keep], tb, [1, 2, 3, 4], want_logits=True)
        assert np.array_equal(ta, tb) and np.array_equal(la, lb)
    for s in [forks[i] for i in keep] + own + [root]:
        s.Close()
    for x in (batch, other):
        x.Close()
    import gc
    gc.collect()  # the fork that was not kept
    assert pool.FreePages == 2 * h * (n + 1)
    pool.Close()
    m.Close()


def test_extend_passes_of_512_tokens(gpu_lib):
    """More tokens than a pass holds, a session's chunk cut by the passes: the
    same caches and scores as in one call per session (the products' sums
    differ in order, so to the bar of the batched paths)."""
    import synthetic
    cfg, m = _load(gpu_lib, "mid")
    ctx = 1024
    batch = gpu_lib.Batch(m, 4)
    chunks = [synthetic.prompt_ids(cfg, k, seed=60 + k) for k in (400, 3, 701)]
    together, alone = [m.NewState(ctx) for _ in chunks], [m.NewState(ctx) for _ in chunks]
    a = batch.extend(together, chunks, targets=chunks, top_k=3)
    b = [batch.extend([s], [c], targets=[c], top_k=3) for s, c in zip(alone, chunks)]
    for k in ("logprob", "entropy", "top_logprobs"):
        x, y = a[k], np.concatenate([r[k] for r in b])
        assert np.linalg.norm(x - y) <= 1e-2 * np.linalg.norm(y), k
    for s, t, c in zip(together, alone, chunks):
        assert s.Pos == t.Pos == len(c)
        for x, y in zip(s.read_kv(0, 0, s.Pos), t.read_kv(0, 0, s.Pos)):
            assert np.linalg.norm(x - y) <= 1e-5 * np.linalg.norm(y)
    for x in together + alone + [batch, m]:
        x.Close()


def test_extend_refusals(gpu_lib):
    cfg, m = _load(gpu_lib, "tiny")
    batch = gpu_lib.Batch(m, 2)
    a, b = m.NewState(32), m.NewState(32)
    E = gpu_lib.L3GError
    batch.extend([a], [[]])  # nothing to do
    for args, kw, msg in ((([a, a], [[1], [2]]), {}, "appears twice"), (([a, b, a], [[1]] * 3), {}, "n=3"),
                          (([a], [[1] * 33]), {}, "context length exceeded"), (([a], [[cfg.vocab]]), {}, "token out"),
                          (([a], [[-1]]), {}, "token out"), (([a], [[1]]), dict(score=True, top_k=65), "top_k"),
                          (([a], [[1, 2]]), dict(targets=[[1]]), "target per token")):
        with pytest.raises(E, match=msg):
            batch.extend(*args, **kw)
    assert a.Pos == b.Pos == 0
    out = batch.extend([a, b], [[1, 2], []], score=True, top_k=2)
    assert out["top_ids"].shape == (2, 2) and "logprob" not in out and a.Pos == 2 and b.Pos == 0
    for x in (a, b, batch, m):
        x.Close()
