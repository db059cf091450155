"""Host-side refusals of the token-level entry points: a status and a message
before any launch (the pointers are never dereferenced)."""
import ctypes

import pytest

P = ctypes.c_void_p(4096)
BIG = 1 << 40
NAN, INF = float("nan"), float("inf")


def _lib():
    from orthocache_b200 import _lib
    return _lib.load()


def _tree(lib, q=P, k=P, dtype=1, table=None, stride=0, pages=0, block=512, dk=P, mask=P, batch=1, nodes=4, hq=8, hkv=2,
          d=128, s=1024, cap=0.0, scale=0.1, out=P, out_dtype=1, ws=P, ws_bytes=BIG):
    return lib.oc_tree_attention(q, k, P, dtype, table, stride, pages, block, None, dk, P, mask, 0, batch, nodes, hq,
                                 hkv, d, s, cap, scale, out, out_dtype, ws, ws_bytes, None)


def _chunk(lib, q=P, k=P, dtype=1, batch=1, n=4, hq=8, hkv=2, d=128, s=1024, cap=0.0, scale=0.1, out=P, out_dtype=1,
           ws=P, ws_bytes=BIG):
    return lib.oc_chunk_attention(q, k, P, dtype, None, 1, None, None, None, batch, n, hq, hkv, d, s, cap, scale, out,
                                  out_dtype, ws, ws_bytes, None)


def _acc(lib, q=P, k=P, dtype=1, w=P, batch=1, n=4, hq=8, hkv=2, d=128, s=1024, cap=0.0, scale=0.1, out=P, out_dtype=1,
         ws=P, ws_bytes=BIG):
    return lib.oc_accumulate_attention(q, k, P, dtype, None, None, w, batch, n, hq, hkv, d, s, cap, scale, out,
                                       out_dtype, ws, ws_bytes, None)


@pytest.mark.parametrize("call", [_tree, _chunk, _acc])
@pytest.mark.parametrize("kw,rc,needle", [
    (dict(q=None), -1, b"NULL"),
    (dict(k=None), -1, b"NULL"),
    (dict(out=None), -1, b"NULL"),
    (dict(dtype=7), -5, b"dtype"),
    (dict(out_dtype=-1), -5, b"dtype"),
    (dict(batch=0), -2, b"batch"),
    (dict(hq=9), -2, b"q_heads"),
    (dict(hkv=0), -2, b"kv_heads"),
    (dict(d=96), -2, b"head_dim"),
    (dict(s=-1), -2, b"seq_len"),
    (dict(batch=1 << 16, s=1 << 16), -2, b"rows"),
    (dict(cap=-2.0), -2, b"cap"),
    (dict(cap=NAN), -2, b"cap"),
    (dict(scale=INF), -2, b"scale"),
    (dict(q=ctypes.c_void_p(4098)), -3, b"aligned"),
    (dict(k=ctypes.c_void_p(4100)), -3, b"aligned"),
    (dict(ws_bytes=0, s=65536), -4, b"workspace"),
])
def test_attention_refusals(call, kw, rc, needle):
    lib = _lib()
    assert call(lib, **kw) == rc
    assert needle in lib.oc_last_error()


@pytest.mark.parametrize("kw,rc,needle", [
    (dict(dk=None), -1, b"NULL"),
    (dict(mask=None), -1, b"NULL"),
    (dict(nodes=0), -2, b"q_len"),
    (dict(nodes=257), -4, b"256"),
    (dict(dk=ctypes.c_void_p(4104)), -3, b"aligned"),
    (dict(table=P, stride=2, pages=4, block=100, s=200), -2, b"block_size"),
    (dict(table=P, stride=2, pages=0), -2, b"num_pages"),
    (dict(table=P, stride=3, pages=4), -2, b"table"),
    (dict(table=P, stride=2, pages=1 << 23), -2, b"pool"),
])
def test_tree_refusals(kw, rc, needle):
    lib = _lib()
    assert _tree(lib, **kw) == rc
    assert needle in lib.oc_last_error()


def test_accumulate_needs_sums():
    lib = _lib()
    assert _acc(lib, w=None) == -1


def test_workspace_query():
    lib = _lib()
    f = lib.oc_token_attention_workspace_bytes
    assert f(1, 1, 0, 8, 2, 128, 100, 0) == 0
    assert f(1, 1, 1, 8, 3, 128, 100, 0) == 0
    assert f(1, 1, 1, 8, 2, 100, 100, 0) == 0
    assert f(1, 1, 1, 8, 2, 128, -1, 0) == 0
    assert f(1, 1, 1, 8, 2, 128, 65536, 0) > 0
    assert f(1, 1, 1, 8, 2, 128, 65536, 1) > f(1, 1, 1, 8, 2, 128, 65536, 0)


@pytest.mark.parametrize("kw,rc,needle", [
    (dict(k=None), -1, b"NULL"),
    (dict(dtype=3), -5, b"dtype"),
    (dict(batch=0), -2, b"batch"),
    (dict(s=0), -2, b"seq_len"),
    (dict(d=12), -2, b"head_dim"),
    (dict(keep=0), -2, b"keep"),
    (dict(keep=101), -2, b"keep"),
    (dict(recent=-1), -2, b"recent"),
    (dict(recent=51), -2, b"recent"),
    (dict(k=ctypes.c_void_p(4100)), -3, b"aligned"),
    (dict(ko=P), -2, b"own"),
])
def test_evict_refusals(kw, rc, needle):
    lib = _lib()
    a = dict(k=P, dtype=1, batch=1, s=100, h=2, d=64, keep=50, recent=10, ko=ctypes.c_void_p(8192))
    a.update(kw)
    got = lib.oc_evict_tokens(a["k"], ctypes.c_void_p(1 << 20), a["dtype"], P, None, a["batch"], a["s"], a["h"],
                              a["d"], a["keep"], a["recent"], a["ko"], ctypes.c_void_p(1 << 21), P, P, P, None)
    assert got == rc
    assert needle in lib.oc_last_error()


@pytest.mark.parametrize("call", [_tree, _chunk, _acc])
@pytest.mark.parametrize("cap,scale", [(1e-30, 0.1), (2e-5, 0.1), (2e-5, -0.1), (1e5, 2e7)])
def test_cap_far_below_the_scale(call, cap, scale):
    """The polynomials of the cap have coefficients up to scale (scale / cap)^8."""
    lib = _lib()
    assert call(lib, cap=cap, scale=scale) == -2
    assert b"scale" in lib.oc_last_error()


@pytest.mark.parametrize("shift", [4, 64, 16 * 1024 - 4, -4])
def test_sums_that_overlap_in_part(shift):
    lib = _lib()  # 1 x 4 heads x 1024 keys x 4 bytes
    w = 1 << 20
    got = lib.oc_accumulate_attention(P, P, P, 1, None, ctypes.c_void_p(w + shift), ctypes.c_void_p(w), 1, 4, 8, 4, 128,
                                      1024, 0.0, 0.1, P, 1, P, BIG, None)
    assert got == -2
    assert b"overlap" in lib.oc_last_error()


def test_evicted_weights_need_a_buffer_of_their_own():
    lib = _lib()
    p = [ctypes.c_void_p(1 << n) for n in range(20, 28)]
    got = lib.oc_evict_tokens(p[0], p[1], 1, p[2], None, 1, 100, 2, 64, 50, 10, p[3], p[4], p[2], p[5], p[6], None)
    assert got == -2
    assert b"own" in lib.oc_last_error()
