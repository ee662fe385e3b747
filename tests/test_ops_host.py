"""Refusals of the serving operators that need no GPU: arguments are checked
before the device is touched."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def l3g():
    import build
    build.build(quiet=True)
    import l3g
    return l3g


@pytest.mark.parametrize("args", [(0, 1, 64, 0), (6, 4, 64, 0), (9, 1, 64, 0), (4, 2, 48, 0), (4, 2, 256, 0),
                                  (4, 2, 64, 2), (4, 2, 64, -1), (-4, -2, 64, 0), (2, 4, 64, 0)])
def test_chunk_attention_shapes(l3g, args):
    with pytest.raises(l3g.L3GError, match="chunk attention|kv_dtype") as e:
        l3g.ChunkAttention(*args)
    assert e.value.code == l3g.L3G_E_INVALID


@pytest.mark.parametrize("args", [(0, 10), (1, 0), (-3, 10), (1, 1 << 25), (1 << 21, 10)])
def test_logprobs_shapes(l3g, args):
    with pytest.raises(l3g.L3GError, match="log probabilities") as e:
        l3g.LogProbs(*args)
    assert e.value.code == l3g.L3G_E_INVALID


def test_null_handles(l3g):
    L = l3g.lib()
    assert L.l3g_chunk_attn_new(4, 2, 64, 0, -1, None) == l3g.L3G_E_INVALID
    assert L.l3g_chunk_attn_run(None, None, 1, 1, None, 256, None, 256, 0, 0.0, None) == l3g.L3G_E_INVALID
    assert L.l3g_chunk_attn_status(None, None, None) == l3g.L3G_E_INVALID
    assert L.l3g_logprobs_new(1, 10, -1, None) == l3g.L3G_E_INVALID
    assert L.l3g_logprobs_run(None, None, 10, 1, None, None, None, None, 0, None, None, None) == l3g.L3G_E_INVALID
    L.l3g_chunk_attn_free(None)
    L.l3g_logprobs_free(None)


def test_copy_pages_arguments(l3g):
    buf = (C.c_uint8 * 4096)()
    base = (C.addressof(buf) + 255) // 256 * 256
    ok = dict(src_pool_ptr=base, n_src=2, dst_pool_ptr=base, n_dst=2, row_bytes=16, src_ptr=base, dst_ptr=base,
              rows_ptr=0, n=1)
    l3g.kv_copy_pages(**{**ok, "n": 0})  # nothing to do
    for change, msg in ((dict(n=-1), "n=-1"), (dict(n_src=-1), "pages"), (dict(row_bytes=0), "rows of"),
                        (dict(row_bytes=24), "rows of"), (dict(row_bytes=1 << 20), "rows of"),
                        (dict(src_pool_ptr=0), "null"), (dict(dst_ptr=0), "null"),
                        (dict(dst_pool_ptr=base + 8), "aligned"), (dict(src_ptr=base + 2), "aligned")):
        with pytest.raises(l3g.L3GError, match=msg):
            l3g.kv_copy_pages(**{**ok, **change})


def test_descriptor_layout(l3g):
    """The binding's descriptor is the header's struct."""
    assert l3g.CHUNK_SEQ.itemsize == 40
    assert [l3g.CHUNK_SEQ.fields[f][1] for f in ("pool", "pages", "n_pages", "pps", "q0", "n_q", "kv_len")] == \
        [0, 8, 16, 20, 24, 28, 32]


def test_state_and_batch_null_arguments(l3g):
    L = l3g.lib()
    out = C.c_void_p()
    n = C.c_int32()
    assert L.l3g_state_fork(None, 0, 0, C.byref(out)) == l3g.L3G_E_INVALID
    assert L.l3g_state_trim(None) == l3g.L3G_E_INVALID
    assert L.l3g_kvpool_compact(None, C.byref(n)) == l3g.L3G_E_INVALID
    assert L.l3g_batch_extend(None, None, 1, None, None, None, None) == l3g.L3G_E_INVALID
    assert L.l3g_logprobs_status(None, None, None) == l3g.L3G_E_INVALID


def test_compaction_moves(tmp_path):
    """compact_plan's rounds put every page in its place through the scratch,
    and no step reads what it writes (tests/pages_plan_check.cpp)."""
    import os
    import subprocess

    from conftest import ROOT
    exe = str(tmp_path / "pages_plan_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I",
                    os.path.join(ROOT, "llama3.go_b200", "csrc"),
                    os.path.join(ROOT, "tests", "pages_plan_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr
