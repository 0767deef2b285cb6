"""CPU tests of what the transformer pieces refuse because two tensors of a call share memory at an offset, before any device
work."""
from __future__ import annotations

import ctypes

import pytest

NULL = ctypes.c_void_p(0)


def at(x, off=0):
    return (x << 32) + off      # addresses far apart, never dereferenced


def vp(x):
    return ctypes.c_void_p(x)


def err(pkg):
    return pkg.lib().tsp_last_error().decode()


# (100 rows of 8 heads of 64 in 16 bits: 102,400 bytes)
@pytest.mark.parametrize("name,kw", [
    ("a row into q", dict(o=at(1, 1024))), ("a head into k", dict(o=at(2, 128))), ("a row into v", dict(o=at(3, 1024))), ("q into out", dict(q=at(4, 1024))),
    ("wider rows over v", dict(o=at(3, 64), o_row=640)), ("q's offsets", dict(qoff=at(4, 2048))), ("k's offsets", dict(koff=at(4, 102396))),
    ("the workspace", dict(ws=at(4, 16))), ("workspace over q", dict(ws=at(1, 16))), ("workspace over k", dict(ws=at(2, 16))),
    ("workspace over v", dict(ws=at(3, 16))), ("workspace over offsets", dict(ws=at(5))),
])
def test_attention(pkg, name, kw):
    L = pkg.lib()
    n, nk, samples = 100, 20_000, 2     # (few rows: split, with a workspace)
    q, k, v = (pkg.Heads(kw.get(x, at(i + 1)), 512, 64) for i, x in enumerate("qkv"))
    o = pkg.Heads(kw.get("o", at(4)), kw.get("o_row", 512), 64)
    need = L.tsp_attention_workspace_bytes(n, nk, samples, 8, 8, 64)
    assert need > 0
    rc = L.tsp_attention(ctypes.byref(q), ctypes.byref(k), ctypes.byref(v), 2, n, nk, 8, 8, 64, vp(kw.get("qoff", at(5))), vp(kw.get("koff", at(6))),
                         samples, 0.125, 0, ctypes.byref(o), vp(kw.get("ws", at(7))), need, NULL)
    assert rc == 1 and ("out must not alias" in err(pkg) or "workspace overlaps" in err(pkg)), (name, rc, err(pkg))


@pytest.mark.parametrize("name,kw", [
    ("q_out a row into k", dict(qo=at(2, 1024))), ("q_out a row into q", dict(qo=at(1, 1024))), ("q_out a head into q", dict(qo=at(1, 128))),
    ("q_out over q with gaps", dict(qo=at(1, 128), qo_row=1024)), ("k_out a head into q", dict(ko=at(1, 128))), ("k_out into k", dict(ko=at(2, 2048))),
    ("k_out into q_out", dict(ko=at(4, 1024))), ("q_out over positions", dict(pos=at(4, 64))), ("k_out over positions", dict(pos=at(5, 64))),
    ("q's factors", dict(gq=at(4, 16))), ("k's factors", dict(gk=at(5, 16))), ("k's factors in q_out", dict(gk=at(4, 16))),
    ("wider values over q", dict(qo=at(1, 102272), odt=0)),
])
def test_rope(pkg, name, kw):
    L = pkg.lib()
    q, k, ko = pkg.Heads(at(1), 512, 64), pkg.Heads(at(2), 512, 64), pkg.Heads(kw.get("ko", at(5)), 512, 64)
    qo = pkg.Heads(kw.get("qo", at(4)), kw.get("qo_row", 512), 64)
    rc = L.tsp_rope_axes(ctypes.byref(q), 8, ctypes.byref(k), 8, 2, 100, 64, vp(kw.get("pos", at(6))), 3, (ctypes.c_int * 3)(10, 10, 10), 1e4, 0,
                         vp(kw.get("gq", at(7))), vp(kw.get("gk", at(8))), 1e-6, ctypes.byref(qo), ctypes.byref(ko), kw.get("odt", 2), NULL)
    assert rc == 1 and "an output overlaps" in err(pkg), (name, rc, err(pkg))
