"""The batched product's activation buffers, used with one layout after
another: where a model's width does not fill the last chunk of columns, the
scales of the padding must be zero whatever the last call left there (a NaN
there spoils a product with zero weights)."""
import numpy as np
import pytest

from conftest import synthetic_model

pytestmark = pytest.mark.gpu


def _load(gpu_lib):
    cfg, T = synthetic_model("tiny-g3")  # n_emb 192: one and a half chunks
    return cfg, gpu_lib.LoadModelFromTensors(gpu_lib.hparams_for(cfg), T,
                                             gpu_lib.default_options(device=0, kv_dtype=0))


def test_prefill_after_another_length(gpu_lib):
    import synthetic
    cfg, m = _load(gpu_lib)
    old, first = m.NewWorkspace(128, 40), None
    for it in range(40):
        a, b = m.NewState(128), m.NewState(128)
        ids = synthetic.prompt_ids(cfg, 128, seed=200 + it)
        m.PrefillBatched(a, ids, old)  # leaves its bytes
        new = m.NewWorkspace(128, 40)
        n = 17 + it % 40
        c, d = m.NewState(128), m.NewState(128)
        m.PrefillBatched(c, ids[:n], old)
        m.PrefillBatched(d, ids[:n], new)
        for layer in range(cfg.n_layers):
            for x, y in zip(c.read_kv(layer, 0, n), d.read_kv(layer, 0, n)):
                assert np.isfinite(x).all() and np.array_equal(x, y), (it, layer)
        for s in (a, b, c, d, new):
            s.Close()
    old.Close()
    m.Close()


def test_batch_step_after_another_size(gpu_lib):
    import synthetic
    cfg, m = _load(gpu_lib)
    old = gpu_lib.Batch(m, 64)
    for it in range(10):
        many = [m.NewState(128) for _ in range(64)]
        ids = synthetic.prompt_ids(cfg, 64, seed=300 + it)
        old.step(many, ids.tolist(), list(range(64)), want_logits=True)
        n = 9 + it
        few = [m.NewState(128) for _ in range(2 * n)]
        new = gpu_lib.Batch(m, 64)
        _, x = old.step(few[:n], ids[:n].tolist(), list(range(n)), want_logits=True)
        _, y = new.step(few[n:], ids[:n].tolist(), list(range(n)), want_logits=True)
        assert np.isfinite(x).all() and np.array_equal(x, y), it
        for s in many + few + [new]:
            s.Close()
    old.Close()
    m.Close()
