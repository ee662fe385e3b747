"""A call that fails with a CUDA error (no memory, no such device) fails alone:
the next call on the thread does not report it again."""
import numpy as np
import pytest

import ops_ref
from conftest import synthetic_model

pytestmark = pytest.mark.gpu


def _logprobs_work(gpu_lib):
    import torch
    op = gpu_lib.LogProbs(2, 500)
    x = np.random.default_rng(1).normal(0, 2, (2, 500)).astype(np.float32)
    xd, td = torch.from_numpy(x).cuda(), torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    lp = torch.zeros(2, device="cuda")

    def call():
        lp.zero_()
        op.run(xd.data_ptr(), 500, 2, td.data_ptr(), lp.data_ptr())
        torch.cuda.synchronize()
        for r, t in enumerate((3, 4)):
            assert abs(lp[r].item() - ops_ref.logprobs(x[r], t, 0)[0]) < 1e-5
    return call


def test_no_memory(gpu_lib):
    call = _logprobs_work(gpu_lib)
    with pytest.raises(gpu_lib.L3GError, match="memory") as e:
        gpu_lib.LogProbs(1 << 20, 1 << 24)  # a terabyte of keys
    assert e.value.code == gpu_lib.L3G_E_CUDA
    call()


def test_no_device(gpu_lib):
    call = _logprobs_work(gpu_lib)
    for make in (lambda: gpu_lib.LogProbs(1, 10, device=63), lambda: gpu_lib.ChunkAttention(2, 1, 64, device=63)):
        with pytest.raises(gpu_lib.L3GError, match="device") as e:
            make()
        assert e.value.code == gpu_lib.L3G_E_CUDA
        call()


def test_no_memory_for_a_pool(gpu_lib):
    cfg, T = synthetic_model("small")
    m = gpu_lib.LoadModelFromTensors(gpu_lib.hparams_for(cfg), T, gpu_lib.default_options(device=0))
    batch = gpu_lib.Batch(m, 2)
    s = m.NewState(64)
    with pytest.raises(gpu_lib.L3GError, match="memory"):
        m.NewKvPool(1 << 24)  # 2 TB
    batch.extend([s], [[1, 2, 3]])
    assert s.Pos == 3
    for x in (s, batch, m):
        x.Close()
