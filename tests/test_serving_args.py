"""Argument checks of the serving-step operators: every refusal comes before
the device is touched (runs without a GPU)."""
import ctypes as C

import pytest

D = C.c_void_p(4096)  # never dereferenced: every check below comes first


@pytest.fixture(scope="module")
def L(mq):
    from minq_b200 import _lib
    return _lib.lib()


def _extend(L, n_req=4, page=16, stride=8, n_pages=32, max_tokens=16, null=None):
    a = dict(lens=D, new=D, table=D, free=D, n_free=D, lo=D, fo=D, qs=D, sl=D, pos=D, info=D)
    if null:
        a[null] = None
    return L.minq_pages_extend(a["lens"], a["new"], n_req, page, a["table"], stride, a["free"],
                               n_pages, a["n_free"], max_tokens, a["lo"], a["fo"], a["qs"], a["sl"],
                               a["pos"], a["info"], None)


def test_pages_refusals(L):
    from minq_b200 import _lib
    for page in (0, 8, 24, 48, 2048):
        assert _extend(L, page=page) == _lib.ERR_SHAPE, page
        assert b"power of two" in L.minq_last_error()
        assert L.minq_pages_trim(D, D, 4, page, D, 8, D, 32, D, D, D, D, None) == _lib.ERR_SHAPE
    assert _extend(L, n_req=8193) == _lib.ERR_SHAPE
    assert _extend(L, stride=0) == _lib.ERR_SHAPE
    assert _extend(L, max_tokens=(1 << 30) + 1) == _lib.ERR_SHAPE
    for null in ("lens", "new", "table", "free", "n_free", "lo", "fo", "qs", "sl", "info"):
        assert _extend(L, null=null) == _lib.ERR_ARG, null
    for i in (0, 1, 4, 6, 8, 9, 10, 11):
        a = [D, D, 4, 16, D, 8, D, 32, D, D, D, D, None]
        a[i] = None
        assert L.minq_pages_trim(*a) == _lib.ERR_ARG, i


def test_kv4_rows_refusals(L):
    from minq_b200 import _lib

    def write(k=D, v=D, ks=1024, vs=1024, slots=D, T=4, nkv=8, hd=128, kp=D, vp=D, n=9, page=16):
        return L.minq_kv4_write(k, v, ks, vs, slots, T, nkv, hd, kp, vp, n, page, None)

    def read(k=D, v=D, ks=1024, vs=1024, slots=D, T=4, nkv=8, hd=128, kp=D, vp=D, n=9, page=16):
        return L.minq_kv4_read(kp, vp, n, page, slots, T, nkv, hd, k, v, ks, vs, None)

    for f in (write, read):
        for hd in (0, 16, 100, 288):
            assert f(hd=hd, ks=8 * 512, vs=8 * 512) == _lib.ERR_SHAPE, hd
        assert f(page=40) == _lib.ERR_SHAPE
        assert f(nkv=0) == _lib.ERR_SHAPE
        assert f(ks=1023) == _lib.ERR_ARG  # tokens would overlap
        assert f(vs=1000) == _lib.ERR_ARG
        for null in ("k", "v", "slots", "kp", "vp"):
            assert f(**{null: None}) == _lib.ERR_ARG, null
        assert f(kp=C.c_void_p(4104)) == _lib.ERR_ARG
        assert b"16-byte aligned" in L.minq_last_error()
        assert f(T=0, k=None, v=None, slots=None) == _lib.OK  # nothing to do


def test_kv4_attend_refusals(L):
    from minq_b200 import _lib

    def attend(q=D, qs=4096, st=D, T=4, lens=D, R=2, table=D, w=8, kp=D, vp=D, n=9, page=16, nh=32,
               nkv=8, hd=128, out=D, os_=4096, ws=D, wb=1 << 40):
        return L.minq_kv4_attend(q, qs, st, T, lens, R, table, w, kp, vp, n, page, nh, nkv, hd, 0.1,
                                 out, os_, ws, wb, None)

    assert attend(nh=30) == _lib.ERR_MODEL
    assert attend(nkv=0) == _lib.ERR_MODEL
    for hd in (0, 80, 288):
        assert attend(hd=hd, qs=1 << 14, os_=1 << 14) == _lib.ERR_SHAPE
    assert attend(page=17) == _lib.ERR_SHAPE
    assert attend(nh=8192) == _lib.ERR_SHAPE
    assert attend(R=8193) == _lib.ERR_SHAPE
    assert attend(T=(1 << 24) + 1) == _lib.ERR_SHAPE
    assert attend(w=0) == _lib.ERR_SHAPE
    assert attend(T=1 << 20, nh=2048, nkv=8, hd=128, qs=1 << 20, os_=1 << 20) == _lib.ERR_SHAPE
    assert attend(qs=4095) == _lib.ERR_ARG
    assert attend(os_=100) == _lib.ERR_ARG
    for null in ("q", "st", "lens", "table", "kp", "vp", "out"):
        assert attend(**{null: None}) == _lib.ERR_ARG, null
    assert attend(vp=C.c_void_p(4100)) == _lib.ERR_ARG
    need = L.minq_kv4_attend_workspace_bytes(2, 4, 32, 8, 128)
    if need:
        assert attend(wb=need - 1) == _lib.ERR_ARG
        assert attend(ws=None, wb=need) == _lib.ERR_ARG
        assert attend(ws=C.c_void_p(4100), wb=need) == _lib.ERR_ARG
    assert attend(T=0, q=None, out=None) == _lib.OK
    assert attend(R=0) == _lib.OK


def test_sample_rows_refusals(L):
    from minq_b200 import _lib

    def rows(x=D, stride=100, r=4, n=100, u=D, out=D):
        return L.minq_sample_rows(x, stride, r, n, None, None, None, None, u, out, None)

    assert rows(n=0) == _lib.ERR_SHAPE
    assert rows(n=(1 << 22) + 1, stride=1 << 23) == _lib.ERR_SHAPE
    assert rows(r=(1 << 20) + 1) == _lib.ERR_SHAPE
    assert rows(stride=99) == _lib.ERR_ARG
    for null in ("x", "u", "out"):
        assert rows(**{null: None}) == _lib.ERR_ARG
    assert rows(r=0, x=None) == _lib.OK


def test_cpu_tensors_are_refused(mq):
    """There is no CPU path: host tensors raise instead of being moved."""
    import torch
    from minq_b200 import _lib
    i = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(2, 1, 16, 40, dtype=torch.uint8)
    s = torch.zeros(1, dtype=torch.int64)
    x = torch.zeros(1, 1, 64)
    for call in (lambda: mq.pages_extend(i, i, i.reshape(2, 1), i, i[:1], 16, 4),
                 lambda: mq.pages_trim(i, i, i.reshape(2, 1), i, i[:1], 16),
                 lambda: mq.kv4_write(x, x, s, pool, pool), lambda: mq.kv4_read(s, pool, pool),
                 lambda: mq.kv4_attend(x, i, i[:1], i.reshape(1, 2), pool, pool),
                 lambda: mq.sample_rows(x[0], x[0, 0, :1])):
        with pytest.raises(mq.MinqError) as e:
            call()
        assert e.value.status == _lib.ERR_CUDA
    with pytest.raises(mq.MinqError):
        mq.kv4_pool(4, 2, 16, 100)
