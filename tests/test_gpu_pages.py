"""Copies between pages of caches (l3g_kv_copy_pages): row counts, row sizes,
two pools, entries outside their bounds, streams."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _ints(torch, a):
    return torch.from_numpy(np.asarray(a, np.int32)).cuda()


@pytest.mark.parametrize("row_bytes,n", [(1024, 5), (128, 40), (16, 3), (512, 700), (48, 9)])
def test_copies_rows(gpu_lib, row_bytes, n):
    import torch
    rng = np.random.default_rng(row_bytes + n)
    a = torch.randint(0, 256, (n + 3, 256, row_bytes), dtype=torch.uint8, device="cuda")
    b = torch.randint(0, 256, (2 * n, 256, row_bytes), dtype=torch.uint8, device="cuda")
    src = rng.integers(0, n + 3, n)  # a source may serve several copies
    dst = rng.permutation(2 * n)[:n]
    rows = rng.integers(0, 257, n)
    rows[:3] = (0, 256, 1)
    want_a, want_b = a.cpu().numpy().copy(), b.cpu().numpy().copy()
    for s, d, r in zip(src, dst, rows):
        want_b[d, :r] = want_a[s, :r]
    st = torch.zeros(2, dtype=torch.int32, device="cuda")
    S, D, R = _ints(torch, src), _ints(torch, dst), _ints(torch, rows)
    gpu_lib.kv_copy_pages(a.data_ptr(), n + 3, b.data_ptr(), 2 * n, row_bytes, S.data_ptr(), D.data_ptr(),
                          R.data_ptr(), n, st.data_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(b.cpu().numpy(), want_b) and np.array_equal(a.cpu().numpy(), want_a)
    assert st.tolist() == [0, 0]


def test_whole_pages_within_one_pool(gpu_lib):
    import torch
    p = torch.randn(64, 256, 2, 64, device="cuda")
    want = p.clone()
    src, dst = list(range(0, 30)), list(range(34, 64))
    want[dst] = want[src]
    S, D = _ints(torch, src), _ints(torch, dst)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gpu_lib.kv_copy_pages(p.data_ptr(), 64, p.data_ptr(), 64, 512, S.data_ptr(), D.data_ptr(), 0, 30,
                          stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(p, want)


@pytest.mark.parametrize("bad", [(-1, 5, 9), (64, 5, 9), (3, -7, 9), (3, 64, 9), (3, 5, -1), (3, 5, 257)])
def test_entries_outside_their_bounds(gpu_lib, bad):
    import torch
    p = torch.randn(64, 256, 32, device="cuda")
    want = p.clone()
    want[40] = want[1]
    want[41, :7] = want[2, :7]
    S, D, R = _ints(torch, [1, bad[0], 2]), _ints(torch, [40, bad[1], 41]), _ints(torch, [256, bad[2], 7])
    st = torch.zeros(2, dtype=torch.int32, device="cuda")
    for status in (st.data_ptr(), 0):
        gpu_lib.kv_copy_pages(p.data_ptr(), 64, p.data_ptr(), 64, 128, S.data_ptr(), D.data_ptr(), R.data_ptr(),
                              3, status)
    torch.cuda.synchronize()
    assert torch.equal(p, want) and st.tolist() == [4, 1]
