"""Infinities in K and q of the chunk attention (l3g_chunk_attn_run) against
the definition in 64 bits: a score of -inf weighs nothing, one of +inf gives
NaN, in the tokens that see the key and in no other."""
import numpy as np
import pytest

import ops_ref
from ops_ref import PAGE, Paged
from test_gpu_chunk_attention import Run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,heads,hkv,n,kv", [(32, 2, 1, 20, 300), (64, 4, 2, 70, 330), (128, 8, 1, 33, 2000),
                                               (128, 4, 1, 1, 5000)])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_infinite_keys(gpu_lib, hd, heads, hkv, n, kv, f16, bad):
    rng = np.random.default_rng(hd + heads)
    cache = Paged(rng, [(kv, 0)], hkv, hd, f16)
    q = rng.normal(0, 1.3, (n, heads, hd)).astype(np.float32)
    q[n // 2, 0, 5] = 0.0     # 0 times infinity: NaN
    q[n // 3, 1, 5] = 1e-9    # far below the row's largest: its sign still counts
    q[n // 4, 1, 5] = -1e-9
    bound = ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))
    run = Run(gpu_lib, cache, [n], heads, q)
    k = cache.k[0].copy()
    for p in (10, kv - n + n // 3, kv - n + n // 2):
        run.pools[0][cache.table[0, 0, p // PAGE], p % PAGE, 0, 5] = bad
        k[0, p, 5] = bad
    run()
    got = run.got()[0]
    assert run.op.status() == (0, 0)
    with np.errstate(invalid="ignore"):
        want = ops_ref.attention(q, (k, cache.v[0]), n, kv)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fin = ~np.isnan(want)
    assert fin.any() and np.abs(got[fin] - want[fin]).max() <= bound


@pytest.mark.parametrize("f16", [False, True])
def test_only_infinite_keys(gpu_lib, f16):
    rng = np.random.default_rng(8)
    n = kv = 140
    cache = Paged(rng, [(kv, 0)], 1, 64, f16)
    q = np.abs(rng.normal(0, 1.3, (n, 2, 64))).astype(np.float32) + 0.1
    run = Run(gpu_lib, cache, [n], 2, q)
    k = cache.k[0].copy()
    page = cache.table[0, 0, 0]
    run.pools[0][page, :70, 0, 4] = -float("inf")
    k[0, :70, 4] = -np.inf
    run.pools[0][page, n - 1, 1, 7] = float("nan")
    run()
    got = run.got()[0]
    assert run.op.status() == (0, 0) and (got[:70] == 0).all()
    want = ops_ref.attention(q[70:-1], (k[:, :-1], cache.v[0][:, :-1]), n - 71, kv - 1)
    assert np.abs(got[70:-1] - want).max() <= ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))
    assert np.isnan(got[-1, :, 7]).all() and np.isfinite(np.delete(got[-1], 7, 1)).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_infinite_query(gpu_lib, f16, bad):
    rng = np.random.default_rng(9)
    n, kv = 40, 700
    cache = Paged(rng, [(kv, 0)], 1, 128, f16)
    q = rng.normal(0, 1.3, (n, 4, 128)).astype(np.float32)
    q[17, 1, 3] = bad
    run = Run(gpu_lib, cache, [n], 4, q)
    run()
    got = run.got()[0]
    assert run.op.status() == (0, 0) and np.isnan(got[17, 1]).all()
    q[17, 1, 3] = 0.0
    want = ops_ref.attention(q, (cache.k[0], cache.v[0]), n, kv)
    got[17, 1] = want[17, 1]
    assert np.abs(got - want).max() <= ops_ref.attention_bound(q, (cache.k[0], cache.v[0]))


@pytest.mark.parametrize("f16", [False, True])
def test_infinite_key_of_a_long_cache(gpu_lib, f16):
    """Every row of many row tiles taken again over 131072 positions, which takes
    longer than other waits of the kernel may: no wait gives up."""
    import torch
    heads, hkv, hd, n, kv = 32, 8, 128, 600, 131072
    g = torch.Generator(device="cuda").manual_seed(1)
    pps = kv // PAGE
    pool = torch.empty(hkv * pps, PAGE, 2, hd, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    for h in range(hkv):
        pool[h * pps:(h + 1) * pps] = torch.randn(pps, PAGE, 2, hd, generator=g, device="cuda")
    pool[::pps, 10, 0, 5] = -float("inf")
    table = torch.arange(hkv * pps, dtype=torch.int32, device="cuda")
    q = torch.randn(n, heads, hd, generator=g, device="cuda") * 1.3
    q[..., 5] = q[..., 5].abs() + 0.01
    out = torch.full_like(q, float("nan"))
    desc = gpu_lib.chunk_seqs(1)
    desc["pool"], desc["n_pages"], desc["pages"], desc["pps"] = pool.data_ptr(), hkv * pps, table.data_ptr(), pps
    desc["n_q"], desc["kv_len"] = n, kv
    sd = torch.from_numpy(desc.view(np.uint8)).cuda()
    op = gpu_lib.ChunkAttention(heads, hkv, hd, gpu_lib.L3G_KV_F16 if f16 else gpu_lib.L3G_KV_F32)
    op.run(sd.data_ptr(), 1, n, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd)
    assert op.status() == (0, 0)
    assert torch.isfinite(out).all()
    for t, h in ((0, 0), (123, 17), (599, 31)):
        cells = pool[h // 4 * pps:(h // 4 + 1) * pps].reshape(kv, 2, hd)
        see = kv - n + t + 1
        K, V = cells[:see, 0].cpu().numpy()[None], cells[:see, 1].cpu().numpy()[None]
        qi = q[t, h].cpu().numpy()[None, None]
        want = ops_ref.attention(qi, (K, V), 1, see)
        K[0, 10, 5] = 0  # (for the bound)
        assert np.abs(out[t, h].cpu().numpy() - want[0, 0]).max() <= ops_ref.attention_bound(qi, (K, V))
