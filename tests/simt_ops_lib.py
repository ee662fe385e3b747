"""ctypes front end of the SIMT emulator build of the serving operators'
kernels (tests/simt/emu_ops.cpp): builds it with g++ on first use.  Test
infrastructure only (CPU tests)."""
import ctypes as C
import os
import subprocess
import tempfile

import numpy as np

from simt_lib import CSRC, ROOT, SIMT, _sources

_lib = None
_P = C.c_void_p


def build():
    out_dir = os.path.join(tempfile.gettempdir(), f"l3g_simt_{os.getuid()}")
    os.makedirs(out_dir, exist_ok=True)
    out = os.path.join(out_dir, "libemu_ops.so")
    if os.path.exists(out) and all(os.path.getmtime(f) <= os.path.getmtime(out) for f in _sources()):
        return out
    cuda_inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    tmp = out + f".{os.getpid()}.tmp"
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-fPIC", "-shared", "-I", cuda_inc,
                    "-I", CSRC, "-I", SIMT, "-I", os.path.join(ROOT, "include"),
                    os.path.join(SIMT, "emu_ops.cpp"), "-o", tmp], check=True)
    os.replace(tmp, out)
    return out


def lib():
    global _lib
    if _lib is None:
        L = C.CDLL(build())
        L.emu_error.restype = C.c_char_p
        L.emu_malloc.restype = _P
        L.emu_malloc.argtypes = [C.c_ulonglong]
        L.emu_free.argtypes = [_P]
        L.emu_schedule.argtypes = [C.c_int, C.c_ulonglong, C.c_int]
        L.emu_chunk_attention.argtypes = [_P, C.c_int, C.c_int, _P, C.c_longlong, _P, C.c_longlong, C.c_int,
                                          C.c_int, C.c_int, C.c_int, C.c_int, C.c_float, C.c_int,
                                          C.POINTER(C.c_int), C.POINTER(C.c_int)]
        L.emu_logprobs.argtypes = [_P, C.c_longlong, C.c_int, C.c_int, _P, _P, _P, _P, C.c_int, _P, _P, C.c_int,
                                   C.c_int, C.POINTER(C.c_int)]
        L.emu_copy_pages.argtypes = [_P, C.c_int, _P, C.c_int, C.c_int, _P, _P, _P, C.c_int, _P, C.c_int]
        _lib = L
    return _lib


class Dev:
    """A device buffer of the emulator holding an array (a guard page after its end)."""

    def __init__(self, arr):
        arr = np.ascontiguousarray(arr)
        self.shape, self.dtype, self.nbytes = arr.shape, arr.dtype, arr.nbytes
        self.ptr = lib().emu_malloc(max(1, self.nbytes))
        if not self.ptr:
            raise RuntimeError(lib().emu_error().decode())
        C.memmove(self.ptr, arr.ctypes.data, self.nbytes)

    def read(self):
        out = np.empty(self.shape, self.dtype)
        C.memmove(out.ctypes.data, self.ptr, self.nbytes)
        return out

    def free(self):
        lib().emu_free(self.ptr)


def check(rc):
    if rc != 0:
        raise RuntimeError(lib().emu_error().decode())


def chunk_attention(cache, chunks, heads, q, grid=3, scale=None, layer=0, seed=None, edit=None, table=None,
                    pools=None, extra=2):
    """Runs the kernels on an ops_ref.Paged cache; returns (out rows, err,
    where).  edit(desc) may change the descriptors, table and pools replace
    the cache's own."""
    import l3g
    L = lib()
    L.emu_schedule(0 if seed is None else 1, seed or 0, 40)
    pool_d = [Dev(p) for p in (pools or cache.pools)]
    table_d = Dev(cache.table if table is None else table)
    desc = l3g.chunk_seqs(len(chunks))
    at = 0
    for i, n in enumerate(chunks):
        p = pool_d[cache.pool_of[i]]
        d = desc[i]
        d["pool"], d["n_pages"] = p.ptr, p.shape[0]
        d["pages"] = table_d.ptr + i * cache.layers * cache.hkv * cache.pps * 4
        d["pps"], d["q0"], d["n_q"], d["kv_len"] = cache.pps, at, n, cache.lens[i]
        at += n
    if edit:
        edit(desc)
    width = heads * cache.hd
    qd = Dev(np.concatenate([q.reshape(at, width), np.full((extra, width), np.nan, np.float32)]))
    out = Dev(np.full((at + extra, width), np.nan, np.float32))
    sd = Dev(desc.view(np.uint8))
    err, where = C.c_int(), C.c_int()
    try:
        check(L.emu_chunk_attention(sd.ptr, len(chunks), at + extra, qd.ptr, width, out.ptr, width, layer, heads,
                                    cache.hkv, cache.hd, int(cache.dt == np.float16),
                                    1.0 / np.sqrt(cache.hd) if scale is None else scale, grid, C.byref(err),
                                    C.byref(where)))
        return out.read(), err.value, where.value
    finally:
        for b in pool_d + [table_d, qd, out, sd]:
            b.free()


def logprobs(x, targets, k, ld=None, shift=0, grid=5, seed=None):
    """Runs the kernels on rows of logits, `shift` floats behind a 16-byte
    boundary at row stride ld; returns a dict of lp, ent, rank, ids, tlp."""
    L = lib()
    L.emu_schedule(0 if seed is None else 1, seed or 0, 40)
    n, v = x.shape
    ld = ld or v
    buf = np.full(shift + n * ld, np.nan, np.float32)
    buf[shift:].reshape(n, ld)[:, :v] = x
    xd, td = Dev(buf), Dev(np.asarray(targets, np.int32))
    o = {"lp": Dev(np.full(n, 7, np.float32)), "ent": Dev(np.full(n, 7, np.float32)),
         "rank": Dev(np.full(n, 7, np.int32)), "ids": Dev(np.full((n, max(k, 1)), 7, np.int32)),
         "tlp": Dev(np.full((n, max(k, 1)), 7, np.float32))}
    err = C.c_int()
    try:
        check(L.emu_logprobs(xd.ptr + 4 * shift, ld, n, v, td.ptr, o["lp"].ptr, o["ent"].ptr, o["rank"].ptr, k,
                             o["ids"].ptr, o["tlp"].ptr, int(shift % 4 == 0 and ld % 4 == 0), grid, C.byref(err)))
        if err.value:
            raise RuntimeError(f"device check {err.value}")
        return {a: b.read() for a, b in o.items()}
    finally:
        for b in [xd, td, *o.values()]:
            b.free()


def copy_pages(src_pool, dst_pool, src, dst, rows=None, max_rows=65535):
    """k_copy_pages between two pools [pages][PAGE][row bytes] (uint8), None for
    dst_pool: within one; returns (the destination pool, status)."""
    L = lib()
    L.emu_schedule(0, 0, 40)
    i32 = np.int32
    a = Dev(src_pool)
    b = a if dst_pool is None else Dev(dst_pool)
    sd, dd, st = Dev(np.asarray(src, i32)), Dev(np.asarray(dst, i32)), Dev(np.zeros(2, i32))
    rd = None if rows is None else Dev(np.asarray(rows, i32))
    try:
        check(L.emu_copy_pages(a.ptr, a.shape[0], b.ptr, b.shape[0], a.shape[2], sd.ptr, dd.ptr,
                               rd.ptr if rd else None, len(src), st.ptr, max_rows))
        return b.read(), tuple(st.read())
    finally:
        for x in {id(y): y for y in (a, b, sd, dd, st, rd) if y}.values():
            x.free()
