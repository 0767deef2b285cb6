"""CPU tests of the transformer pieces' boundary: arguments are refused with a status and a message before
any device work, empty calls are no-ops, and the Python calls refuse what the kernels could not read."""
from __future__ import annotations

import ctypes
import math

import pytest

FAKE = ctypes.c_void_p(0x1000)   # never dereferenced
NULL = ctypes.c_void_p(0)


def _err(pkg):
    return pkg.lib().tsp_last_error().decode()


def test_group_norm_refusals(pkg):
    L = pkg.lib()

    def f(**kw):
        return L.tsp_group_norm(kw.get("x", FAKE), kw.get("xdt", 0), kw.get("n", 100), kw.get("c", 64), kw.get("g", 8),
                                kw.get("off", FAKE), kw.get("samples", 2), NULL, NULL, kw.get("eps", 1e-6), 0,
                                kw.get("out", ctypes.c_void_p(0x2000)), kw.get("odt", 0), kw.get("ws", FAKE), kw.get("wsb", 1 << 20), NULL)
    assert f(n=-1) == 1 and f(n=1 << 31) == 1 and f(c=0) == 1 and "out of range" in _err(pkg)
    assert f(g=0) == 1 and f(g=7) == 1 and "groups" in _err(pkg)
    assert f(samples=0) == 1 and f(off=NULL) == 1 and "samples" in _err(pkg)
    assert f(xdt=3) == 1 and f(odt=-1) == 1 and f(eps=-1.0) == 1 and f(eps=math.nan) == 1
    assert f(c=8192, g=8192) == 4
    assert f(x=NULL) == 1 and f(out=NULL) == 1 and f(ws=NULL) == 1
    assert f(out=FAKE, odt=2) == 1 and "in place" in _err(pkg)
    assert f(ws=ctypes.c_void_p(0x1004)) == 1 and "aligned" in _err(pkg)
    need = L.tsp_group_norm_workspace_bytes(100, 64, 8, 2)
    assert need > 0 and f(wsb=need - 1) == 5 and "workspace" in _err(pkg)
    assert f(n=0, x=NULL, ws=NULL, wsb=0) == 0
    assert L.tsp_group_norm_workspace_bytes(-1, 64, 8, 1) == 0 and L.tsp_group_norm_workspace_bytes(5, 64, 0, 1) == 0
    assert f(samples=(1 << 31) - 1, wsb=(1 << 63)) == 1


def _heads(pkg, data=0x10000, row=512, head=64):
    return pkg.Heads(data, row, head)


def test_rope_refusals(pkg):
    L = pkg.lib()

    def f(**kw):
        q, k = kw.get("q", _heads(pkg)), kw.get("k", _heads(pkg, 0x20000))
        qo, ko = kw.get("qo", _heads(pkg, 0x30000)), kw.get("ko", _heads(pkg, 0x40000))
        pairs = kw.get("pairs", [10, 10, 10])
        ref = lambda h: None if h is None else ctypes.byref(h)
        return L.tsp_rope_axes(ref(q), kw.get("hq", 8), ref(k), kw.get("hk", 8), kw.get("dt", 2), kw.get("n", 100), kw.get("d", 64),
                               kw.get("pos", FAKE), kw.get("axes", 3), (ctypes.c_int * len(pairs))(*pairs), kw.get("theta", 1e4),
                               kw.get("flags", 0), kw.get("gq", NULL), kw.get("gk", NULL), kw.get("eps", 1e-6), ref(qo), ref(ko), kw.get("odt", 2), NULL)
    assert f(n=-1) == 1 and f(n=1 << 31) == 1 and f(dt=5) == 1 and f(odt=3) == 1 and f(flags=2) == 1
    assert f(hq=0) == 1 and f(hk=-1) == 1 and f(hk=0) == 1 and f(k=None) == 1 and f(hq=4096) == 1
    assert f(d=60) == 4 and f(d=264) == 4 and f(d=0) == 4 and "multiple of 8" in _err(pkg)
    assert f(axes=0) == 1 and f(axes=5, pairs=[1] * 5) == 1
    assert f(pairs=[-1, 2, 2]) == 1 and f(pairs=[11, 11, 11]) == 1 and "pairs" in _err(pkg)
    assert f(theta=0.0) == 1 and f(theta=math.inf) == 1 and f(eps=-1.0) == 1 and f(eps=math.nan) == 1
    assert f(q=None) == 1 and f(qo=None) == 1 and f(pos=NULL) == 1 and f(ko=None) == 1 and f(q=_heads(pkg, 0)) == 1
    assert f(q=_heads(pkg, 0x10008)) == 1 and f(q=_heads(pkg, row=516)) == 1 and f(k=_heads(pkg, row=1 << 21)) == 1
    assert f(qo=_heads(pkg, 0x30000, 256, 64)) == 1 and f(ko=_heads(pkg, 0x30000, 512, 32)) == 1 and "overlap" in _err(pkg)
    assert f(gq=ctypes.c_void_p(0x1004)) == 1 and f(gk=ctypes.c_void_p(0x1008)) == 1 and "gamma" in _err(pkg)
    # an output that is another tensor of the call, or its own input seen differently
    assert f(qo=_heads(pkg, 0x20000)) == 1 and f(ko=_heads(pkg, 0x10000)) == 1 and f(ko=_heads(pkg, 0x30000)) == 1
    assert f(qo=_heads(pkg, 0x10000), odt=0) == 1 and f(ko=_heads(pkg, 0x20000, 1024, 64)) == 1
    assert f(qo=_heads(pkg, 0x10000, 64, 6400)) == 1 and "its own input" in _err(pkg)
    assert f(n=0, q=None, pos=NULL) == 0
    assert f(n=0, q=None, pos=NULL, k=None, hk=0) == 0


def test_attention_refusals(pkg):
    L = pkg.lib()

    def f(**kw):
        q, k, v, o = (kw.get(name, _heads(pkg, 0x10000 * (i + 1))) for i, name in enumerate(("q", "k", "v", "o")))
        ref = lambda h: None if h is None else ctypes.byref(h)
        return L.tsp_attention(ref(q), ref(k), ref(v), kw.get("dt", 2), kw.get("nq", 100), kw.get("nk", 100), kw.get("hq", 8),
                               kw.get("hkv", 8), kw.get("d", 64), kw.get("qoff", FAKE), kw.get("koff", FAKE), kw.get("samples", 2),
                               kw.get("scale", 0.125), 0, ref(o), kw.get("ws", FAKE), kw.get("wsb", 1 << 62), NULL)
    assert f(nq=-1) == 1 and f(nk=-1) == 1 and f(nq=1 << 31) == 1 and f(nk=(1 << 31) - 1) == 1
    assert f(hq=0) == 1 and f(hkv=0) == 1 and f(hkv=3) == 1 and f(hq=4, hkv=8) == 1 and "heads" in _err(pkg)
    assert f(dt=3) == 1 and f(dt=-1) == 1 and f(d=60) == 4 and f(d=136) == 4 and f(d=-8) == 4
    assert f(samples=0) == 1 and f(qoff=NULL) == 1 and f(koff=NULL) == 1
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert f(scale=scale) == 1
    assert f(q=None) == 1 and f(o=None) == 1 and f(k=None) == 1 and f(v=_heads(pkg, 0)) == 1
    assert f(q=_heads(pkg, 0x10008)) == 1 and f(k=_heads(pkg, 0x20000, 514)) == 1 and f(v=_heads(pkg, 0x30000, 1 << 21)) == 1
    assert f(o=_heads(pkg, 0x40000, 256)) == 1 and "overlap" in _err(pkg)
    assert f(k=_heads(pkg, 0x20000, 0)) == 1 and f(v=_heads(pkg, 0x30000, 56), nk=1) == 1 and "rows overlap" in _err(pkg)
    assert f(o=_heads(pkg, 0x10000)) == 1 and "alias" in _err(pkg)
    assert f(nq=0, q=None, o=None) == 0
    # one token against a long cache: its keys are split, whatever the mask and type
    assert L.tsp_attention_workspace_bytes(1, 100_000, 1, 16, 2, 128) > 1 << 16
    few = dict(nq=1, nk=100_000, hq=16, hkv=2, d=128, samples=1, q=_heads(pkg, 0x10000, 2048, 128), k=_heads(pkg, 0x20000, 256, 128),
               v=_heads(pkg, 0x30000, 256, 128), o=_heads(pkg, 0x40000, 2048, 128))
    for dt in (0, 1, 2):
        assert f(dt=dt, wsb=1024, **few) == 5 and "workspace" in _err(pkg)
        assert f(dt=dt, ws=NULL, **few) == 1 and "null workspace" in _err(pkg)
        assert f(dt=dt, ws=ctypes.c_void_p(0x1008), **few) == 1 and "aligned" in _err(pkg)
    assert L.tsp_attention_workspace_bytes(0, 5, 1, 8, 8, 64) == 0 and L.tsp_attention_workspace_bytes(5, 5, 1, 8, 3, 64) == 0


def test_python_refusals(pkg):
    import torch
    x, pos = torch.zeros(4, 16), torch.zeros(4, 3, dtype=torch.int32)
    q = torch.zeros(4, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        pkg.group_norm(x, 4)
    with pytest.raises(ValueError, match="multiple of groups"):
        pkg.group_norm(x, 3)
    with pytest.raises(ValueError, match="int32"):
        pkg.group_norm(x, 4, offsets=torch.zeros(3))
    with pytest.raises(ValueError, match="gamma"):
        pkg.group_norm(x, 4, gamma=torch.zeros(15))
    with pytest.raises(ValueError, match="shape"):
        pkg.group_norm(x, 4, out=torch.zeros(4, 15))
    with pytest.raises(ValueError, match="GPU"):
        pkg.rope_axes(q, pos)
    with pytest.raises(ValueError, match="pos"):
        pkg.rope_axes(q, pos.long())
    with pytest.raises(ValueError, match="axes"):
        pkg.rope_axes(q, pos, pairs=[2, 2])
    with pytest.raises(ValueError, match="k_gamma"):
        pkg.rope_axes(q, pos, k_gamma=torch.zeros(2, 16))
    with pytest.raises(ValueError, match="q_gamma"):
        pkg.rope_axes(q, pos, q_gamma=torch.zeros(16))
    with pytest.raises(ValueError, match="one dtype"):
        pkg.rope_axes(q, pos, k=q.half())
    with pytest.raises(ValueError, match="GPU"):
        pkg.attention(q, q, q)
    with pytest.raises(ValueError, match="come together"):
        pkg.attention(q, q, q, q_offsets=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="same samples"):
        pkg.attention(q, q, q, torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="one dtype"):
        pkg.attention(q, q.half(), q)
    with pytest.raises(ValueError, match="must be \\["):
        pkg.attention(q, q, q[:2])
