"""CPU tests of the served block's boundary: arguments are refused with a status and a message before any device work, empty
calls are no-ops, sizes are what the layouts say, and the Python calls refuse what the kernels could not read."""
from __future__ import annotations

import ctypes
import math

import pytest

NULL = ctypes.c_void_p(0)


def at(x):
    return ctypes.c_void_p(x << 32)      # addresses far apart, never dereferenced


def _err(pkg):
    return pkg.lib().tsp_last_error().decode()


def test_rms_norm_refusals(pkg):
    L = pkg.lib()

    def f(**kw):
        return L.tsp_rms_norm(kw.get("x", at(1)), kw.get("xdt", 2), kw.get("n", 10), kw.get("c", 64), kw.get("r", at(2)), kw.get("rdt", 0),
                              kw.get("g", at(3)), kw.get("eps", 1e-6), kw.get("out", at(4)), kw.get("odt", 2), kw.get("p", at(5)),
                              kw.get("ro", at(6)), NULL)
    assert f(n=-1) == 1 and f(n=1 << 31) == 1 and f(c=0) == 1 and f(c=(1 << 20) + 1) == 1 and "out of range" in _err(pkg)
    assert f(xdt=3) == 1 and f(rdt=4) == 1 and f(odt=4) == 1 and f(odt=-1) == 1 and "dtype" in _err(pkg)
    assert f(eps=-1.0) == 1 and f(eps=math.nan) == 1 and f(eps=math.inf) == 1
    assert f(odt=pkg.TSP_MX8, c=48) == 4 and "multiple of 32" in _err(pkg)
    assert f(r=NULL) == 1 and "without a residual" in _err(pkg)
    assert f(x=NULL) == 1 and f(out=NULL) == 1 and f(odt=pkg.TSP_MX8, p=NULL) == 1 and "null" in _err(pkg)
    # an output may be an input of its dtype, and overlap nothing otherwise
    part = ctypes.c_void_p((1 << 32) + 16)
    assert f(out=part) == 1 and f(out=at(1), odt=0) == 1 and f(out=at(2)) == 1 and f(ro=part) == 1 and "overlaps an input" in _err(pkg)
    assert f(odt=pkg.TSP_MX8, p=at(1)) == 1 and f(odt=pkg.TSP_MX8, out=at(1)) == 1
    assert f(out=at(6), odt=0) == 1 and f(out=at(3)) == 1 and f(ro=at(3)) == 1 and f(odt=pkg.TSP_MX8, p=at(4)) == 1 and "each other" in _err(pkg)
    assert f(n=0, x=NULL, out=NULL) == 0


def test_mx_quantize_refusals(pkg):
    L = pkg.lib()

    def f(**kw):
        return L.tsp_mx_quantize(kw.get("x", at(1)), kw.get("dt", 2), kw.get("n", 10), kw.get("c", 64), kw.get("q", at(2)), kw.get("p", at(3)), NULL)
    assert f(n=-1) == 1 and f(c=0) == 1 and f(dt=3) == 1 and f(c=40) == 4 and "multiple of 32" in _err(pkg)
    assert f(x=NULL) == 1 and f(q=NULL) == 1 and f(p=NULL) == 1
    assert f(x=ctypes.c_void_p(0x1008)) == 1 and f(q=ctypes.c_void_p(0x1004)) == 1 and "aligned" in _err(pkg)
    assert f(q=at(1)) == 1 and f(p=at(1)) == 1 and f(p=at(2)) == 1 and "overlap" in _err(pkg)
    assert f(n=0, x=NULL) == 0


def test_linear_mx_refusals(pkg):
    L = pkg.lib()

    def f(**kw):
        return L.tsp_linear_mx(kw.get("x", at(1)), kw.get("xp", at(2)), kw.get("n", 10), kw.get("ci", 64), kw.get("w", at(3)), kw.get("wp", at(4)),
                               kw.get("b", at(5)), kw.get("co", 20), kw.get("act", 0), kw.get("r", at(6)), kw.get("out", at(7)), kw.get("odt", 0),
                               kw.get("ws", at(8)), kw.get("wsb", 1 << 40), NULL)
    assert f(n=-1) == 1 and f(n=1 << 31) == 1 and f(ci=0) == 1 and f(co=0) == 1 and f(ci=1 << 21) == 1 and "out of range" in _err(pkg)
    assert f(odt=3) == 1 and f(act=2) == 1 and f(act=-1) == 1
    assert f(ci=48) == 4 and "multiple of 32" in _err(pkg)
    for name in ("x", "xp", "w", "wp", "out"):
        assert f(**{name: NULL}) == 1 and "null" in _err(pkg)
    for name, p in (("x", 0x1008), ("w", 0x1008), ("xp", 0x1002), ("wp", 0x1001)):
        assert f(**{name: ctypes.c_void_p(p)}) == 1 and "aligned" in _err(pkg)
    for i in range(1, 6):
        assert f(out=at(i)) == 1 and "overlaps" in _err(pkg)
    assert f(out=at(6), odt=2) == 1 and f(out=ctypes.c_void_p((6 << 32) + 4)) == 1
    assert f(n=0, x=NULL) == 0
    assert L.tsp_linear_mx_workspace_bytes(-1, 64, 64) == 0 and L.tsp_linear_mx_workspace_bytes(5, 0, 64) == 0


def heads(pkg, data, row=512, head=64):
    return pkg.Heads(data << 32 if data < 1 << 32 else data, row, head)


def ref(h):
    return None if h is None else ctypes.byref(h)


def cache_arg(pkg, **kw):
    return pkg.KvCacheArg(kw.get("data", 9 << 32), kw.get("pages", 100), kw.get("page", 16), kw.get("heads", 8), kw.get("d", 64),
                          kw.get("format", pkg.TSP_KV_MX4))


BAD_CACHES = [dict(page=8), dict(page=24), dict(page=512), dict(page=0), dict(heads=0), dict(d=60), dict(d=136), dict(d=0), dict(format=0), dict(format=3),
              dict(pages=-1), dict(pages=1 << 31)]


def test_page_bytes(pkg):
    f = pkg.lib().tsp_kv_page_bytes
    assert f(64, 4, 128, pkg.TSP_KV_MX4) == 64 * 4 * 2 * (64 + 4)
    assert f(16, 3, 80, pkg.TSP_KV_MX4) == 16 * 3 * 2 * (48 + 3)
    assert f(32, 2, 72, pkg.TSP_BF16) == 32 * 2 * 2 * 72 * 2
    assert f(15, 2, 64, pkg.TSP_BF16) == 0 and f(16, 2, 64, pkg.TSP_F32) == 0 and f(16, 2, 12, pkg.TSP_F16) == 0


def test_kv_append_refusals(pkg):
    L = pkg.lib()

    def f(cache=None, **kw):
        q, k, v, qo = (kw.get(name, heads(pkg, i + 1)) for i, name in enumerate(("q", "k", "v", "qo")))
        pairs = kw.get("pairs", [10, 10, 10])
        c = cache_arg(pkg, **(cache or {}))
        return L.tsp_kv_append(None if kw.get("nocache") else ctypes.byref(c), ref(k), ref(v), kw.get("dt", 2), kw.get("n", 100), kw.get("off", at(5)),
                               kw.get("samples", 2), kw.get("table", at(6)), kw.get("mp", 7), kw.get("len", at(7)), ref(q), kw.get("hq", 8),
                               kw.get("pos", at(8)), kw.get("axes", 3), (ctypes.c_int * len(pairs))(*pairs), kw.get("theta", 1e4), kw.get("flags", 0),
                               kw.get("gq", NULL), kw.get("gk", NULL), kw.get("eps", 1e-6), ref(qo), NULL)
    for bad in BAD_CACHES:
        assert f(bad) == 4 and "cache" in _err(pkg), bad
    assert f(nocache=True) == 1
    assert f(n=-1) == 1 and f(n=1 << 31) == 1 and f(dt=3) == 1 and f(samples=0) == 1 and f(off=NULL) == 1 and f(mp=0) == 1 and f(flags=2) == 1
    assert f(hq=0) == 1 and f(hq=-1) == 1 and f(hq=4097) == 1 and f(q=None) == 1 and f(qo=None) == 1
    assert f(axes=-1) == 1 and f(axes=5, pairs=[1] * 5) == 1 and f(pairs=[-1, 2, 2]) == 1 and f(pairs=[11, 11, 11]) == 1 and "pairs" in _err(pkg)
    assert f(theta=0.0) == 1 and f(theta=math.inf) == 1 and f(eps=-1.0) == 1 and f(eps=math.nan) == 1
    assert f(k=None) == 1 and f(v=None) == 1 and f(table=NULL) == 1 and f(len=NULL) == 1 and f(pos=NULL) == 1 and f(dict(data=0)) == 1
    assert f(k=heads(pkg, 2, 514)) == 1 and f(v=heads(pkg, (3 << 32) + 8)) == 1 and f(q=heads(pkg, 1, 1 << 21)) == 1 and f(dict(data=(9 << 32) + 8)) == 1
    assert f(gq=ctypes.c_void_p(0x1004)) == 1 and f(gk=ctypes.c_void_p(0x1008)) == 1 and "aligned" in _err(pkg)
    assert f(k=heads(pkg, 9)) == 1 and f(v=heads(pkg, 9)) == 1 and f(qo=heads(pkg, 9)) == 1 and f(q=heads(pkg, 9)) == 1
    assert f(qo=heads(pkg, 4, 256)) == 1 and "overlap" in _err(pkg)
    assert f(qo=heads(pkg, 2)) == 1 and f(qo=heads(pkg, 3)) == 1 and f(qo=heads(pkg, 1, 1024)) == 1 and "may be q" in _err(pkg)
    assert f(n=0, k=None, v=None, table=NULL) == 0


def test_kv_gather_refusals(pkg):
    L = pkg.lib()

    def f(cache=None, **kw):
        k, v = kw.get("k", heads(pkg, 1)), kw.get("v", heads(pkg, 2))
        c = cache_arg(pkg, **(cache or {}))
        return L.tsp_kv_gather(None if kw.get("nocache") else ctypes.byref(c), kw.get("n", 100), kw.get("off", at(5)), kw.get("samples", 2),
                               kw.get("table", at(6)), kw.get("mp", 7), kw.get("len", at(7)), ref(k), ref(v), kw.get("dt", 2), NULL)
    for bad in BAD_CACHES:
        assert f(bad) == 4 and "cache" in _err(pkg), bad
    assert f(nocache=True) == 1 and f(n=-1) == 1 and f(dt=3) == 1 and f(samples=0) == 1 and f(off=NULL) == 1 and f(mp=0) == 1
    assert f(k=None) == 1 and f(v=None) == 1 and f(table=NULL) == 1 and f(len=NULL) == 1 and f(dict(data=0)) == 1
    assert f(k=heads(pkg, 1, 516)) == 1 and f(k=heads(pkg, 1, 256)) == 1 and f(v=heads(pkg, 1)) == 1 and f(k=heads(pkg, 9)) == 1 and f(v=heads(pkg, 9)) == 1
    assert f(n=0, k=None, v=None) == 0


def test_attention_cached_refusals(pkg):
    L = pkg.lib()

    def f(cache=None, **kw):
        q, o = kw.get("q", heads(pkg, 1)), kw.get("o", heads(pkg, 2))
        c = cache_arg(pkg, **(cache or {}))
        return L.tsp_attention_cached(ref(q), kw.get("dt", 2), kw.get("nq", 100), kw.get("hq", 8), None if kw.get("nocache") else ctypes.byref(c),
                                      kw.get("off", at(5)), kw.get("samples", 2), kw.get("table", at(6)), kw.get("mp", 7), kw.get("len", at(7)),
                                      kw.get("scale", 0.125), 1, ref(o), kw.get("ws", at(8)), kw.get("wsb", 1 << 62), NULL)
    for bad in BAD_CACHES:
        assert f(bad) == 4 and "cache" in _err(pkg), bad
    assert f(nocache=True) == 1 and f(dt=0) == 4 and f(dt=3) == 1 and f(dict(format=pkg.TSP_F16)) == 4 and "dtype" in _err(pkg)
    assert f(nq=-1) == 1 and f(nq=1 << 31) == 1 and f(hq=0) == 1 and f(hq=12) == 1 and f(hq=8192) == 1 and f(samples=0) == 1 and f(off=NULL) == 1
    assert f(mp=0) == 1 and f(mp=1 << 28) == 1
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert f(scale=scale) == 1
    assert f(q=None) == 1 and f(o=None) == 1 and f(table=NULL) == 1 and f(len=NULL) == 1 and f(dict(data=0)) == 1
    assert f(q=heads(pkg, 1, 516)) == 1 and f(o=heads(pkg, (2 << 32) + 8)) == 1 and f(o=heads(pkg, 2, 256)) == 1
    assert f(o=heads(pkg, 1)) == 1 and f(o=heads(pkg, 9)) == 1 and "alias" in _err(pkg)
    c = cache_arg(pkg)
    need = L.tsp_attention_cached_workspace_bytes(100, 2, 8, ctypes.byref(c), 7)
    assert need > 0 and f(wsb=need - 1) == 5 and f(ws=NULL) == 1 and f(ws=ctypes.c_void_p((8 << 32) + 8)) == 1
    assert L.tsp_attention_cached_workspace_bytes(0, 2, 8, ctypes.byref(c), 7) == 0
    assert L.tsp_attention_cached_workspace_bytes(100, 2, 9, ctypes.byref(c), 7) == 0
    assert f(nq=0, q=None, o=None) == 0


def test_python_refusals(pkg):
    import torch
    x = torch.zeros(4, 64)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    mx = pkg.mx_empty(4, 64, "cpu")
    for match, call in [
        ("GPU", lambda: pkg.rms_norm(x)), ("gamma", lambda: pkg.rms_norm(x, torch.zeros(63))), ("residual must", lambda: pkg.rms_norm(x, residual=x[:2])),
        ("needs a residual", lambda: pkg.rms_norm(x, residual_out=x)), ("GPU|live on", lambda: pkg.rms_norm(x, residual=x, residual_out=x)),
        ("must be \\[N, C\\]", lambda: pkg.rms_norm(x[0])),
        ("multiple of 32", lambda: pkg.mx_empty(4, 40, "cpu")), ("multiple of 32", lambda: pkg.mx_quantize(x[:, :40])), ("GPU", lambda: pkg.mx_quantize(x)),
        ("GPU", lambda: pkg.linear_mx(mx, mx)), ("must be Mx", lambda: pkg.linear_mx((x, x), mx)), ("codes", lambda: pkg.linear_mx((mx.codes[:3], mx.powers), mx)),
        ("16, 32", lambda: pkg.kv_cache(2, 24, 1, 64, device="cpu")), ("holds", lambda: pkg.kv_cache(2, 16, 1, 64, torch.float32, "cpu")),
        ("data must", lambda: pkg.KVCache(torch.zeros(2, 5, dtype=torch.uint8), 16, 1, 64, "mx4")),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    cache = pkg.kv_cache(4, 16, 2, 64, device="cpu")
    assert cache.data.shape == (4, 16 * 2 * 2 * 34) and cache.pages == 4
    k, q, table, lengths = torch.zeros(3, 2, 64), torch.zeros(3, 4, 64).half(), i32(1, 2), i32(1)
    for match, call in [
        ("GPU", lambda: pkg.kv_append(cache, k, k, table, lengths)), ("must be", lambda: pkg.kv_append(cache, k, k[:2], table, lengths)),
        ("one dtype", lambda: pkg.kv_append(cache, k, k.half(), table, lengths)), ("one dtype", lambda: pkg.kv_append(cache, k, k, table, lengths, q=q)),
        ("need q", lambda: pkg.kv_append(cache, k, k, table, lengths, q_gamma=k)), ("table", lambda: pkg.kv_append(cache, k, k, table.long(), lengths)),
        ("table", lambda: pkg.kv_append(cache, k, k, table, lengths, offsets=i32(3))), ("lengths", lambda: pkg.kv_append(cache, k, k, table, i32(2))),
        ("int32", lambda: pkg.kv_append(cache, k, k, table, lengths, offsets=torch.zeros(2))),
        ("rows", lambda: pkg.kv_gather(cache, table, lengths)), ("GPU", lambda: pkg.kv_gather(cache, table, lengths, n=3)),
        ("GPU", lambda: pkg.attention_cached(q, cache, table, lengths)), ("float16 or", lambda: pkg.attention_cached(q.float(), cache, table, lengths)),
        ("multiple of", lambda: pkg.attention_cached(q[:, :3], cache, table, lengths)),
        ("16-bit cache", lambda: pkg.attention_cached(q, pkg.kv_cache(4, 16, 2, 64, torch.bfloat16, "cpu"), table, lengths)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
