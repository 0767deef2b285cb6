"""CPU tests of what the served block's calls refuse because two of their tensors share memory: the comparison itself against a
byte-by-byte one, and each call's outputs over its inputs at an offset, before any device work."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL = ctypes.c_void_p(0)


def at(x, off=0):
    return (x << 32) + off      # addresses far apart, never dereferenced


def vp(x):
    return ctypes.c_void_p(x)


def err(pkg):
    return pkg.lib().tsp_last_error().decode()


def test_comparison(tmp_path):
    exe = str(tmp_path / "overlap_check")
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                        "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "trellis.cpp_amd", "csrc"), "-o", exe,
                        os.path.join(ROOT, "tests", "host", "overlap_check.cpp")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr[-3000:]


def cache_arg(pkg, data=at(9)):
    return pkg.KvCacheArg(data, 100, 16, 8, 64, pkg.TSP_KV_MX4)


# (100 rows of 8 heads of 64 in 16 bits: 102,400 bytes)
@pytest.mark.parametrize("name,kw", [
    ("a row into q", dict(o=at(1, 1024))), ("a head into q", dict(o=at(1, 128))), ("q a row into out", dict(q=at(2, 1024))),
    ("q's last head", dict(o=at(1, 102400 - 128))), ("wide rows over q", dict(o=at(1, 64), o_row=640)),
    ("the table", dict(table=at(2, 1024))), ("lengths", dict(lengths=at(2, 102396))), ("offsets", dict(off=at(2))),
    ("the workspace", dict(ws=at(2, 16))), ("the cache", dict(o=at(9, 4096))),
    ("workspace over q", dict(ws=at(1, 16))), ("workspace over the table", dict(table=at(8, 64))), ("workspace over lengths", dict(lengths=at(8, 64))),
    ("workspace over offsets", dict(off=at(8, 64))), ("workspace over the cache", dict(ws=at(9, 64))),
])
def test_attention_cached(pkg, name, kw):
    L = pkg.lib()
    q, o = pkg.Heads(kw.get("q", at(1)), 512, 64), pkg.Heads(kw.get("o", at(2)), kw.get("o_row", 512), 64)
    c = cache_arg(pkg)
    ws = kw.get("ws", at(8))
    need = L.tsp_attention_cached_workspace_bytes(100, 2, 8, ctypes.byref(c), 7)
    rc = L.tsp_attention_cached(ctypes.byref(q), 2, 100, 8, ctypes.byref(c), vp(kw.get("off", at(5))), 2, vp(kw.get("table", at(6))), 7,
                                vp(kw.get("lengths", at(7))), 0.125, 1, ctypes.byref(o), vp(ws), need, NULL)
    assert rc == 1 and ("alias" in err(pkg) or "workspace overlaps" in err(pkg)), (name, rc)


@pytest.mark.parametrize("name,kw", [
    ("values a row into keys", dict(v=at(1, 1024))), ("a head", dict(v=at(1, 128))), ("keys into values", dict(k=at(2, 51200))),
    ("wider rows", dict(v=at(1, 1024), v_row=1024)), ("the table", dict(table=at(1, 2048))), ("lengths", dict(lengths=at(2))),
    ("offsets", dict(off=at(2, 102396))), ("the cache", dict(k=at(9, 4096))),
])
def test_kv_gather(pkg, name, kw):
    L = pkg.lib()
    k, v = pkg.Heads(kw.get("k", at(1)), 512, 64), pkg.Heads(kw.get("v", at(2)), kw.get("v_row", 512), 64)
    c = cache_arg(pkg)
    rc = L.tsp_kv_gather(ctypes.byref(c), 100, vp(kw.get("off", at(5))), 2, vp(kw.get("table", at(6))), 7, vp(kw.get("lengths", at(7))),
                         ctypes.byref(k), ctypes.byref(v), 2, NULL)
    assert rc == 1 and "overlap" in err(pkg), (name, rc)


@pytest.mark.parametrize("name,kw", [
    ("q_out a row into k", dict(qo=at(2, 1024))), ("q_out a head into v", dict(qo=at(3, 128))), ("k a row into q_out", dict(k=at(4, 1024))),
    ("q_out a row into q", dict(qo=at(1, 1024))), ("q_out a head into q", dict(qo=at(1, 128))), ("q's rows with gaps", dict(qo=at(1, 128), qo_row=1024)),
    ("the table", dict(table=at(4, 2048))), ("lengths", dict(lengths=at(4))), ("offsets", dict(off=at(4, 102396))), ("positions", dict(pos=at(4, 64))),
    ("q's factors", dict(gq=at(4, 16))), ("k's factors", dict(gk=at(4, 16))), ("the cache", dict(qo=at(9, 4096))),
    ("the cache over k", dict(k=at(9, 4096))), ("... v", dict(v=at(9, 4096))), ("... q", dict(q=at(9, 4096), qo=at(9, 4096))),
    ("... the table", dict(table=at(9, 64))), ("... lengths", dict(lengths=at(9))), ("... offsets", dict(off=at(9))), ("... positions", dict(pos=at(9))),
    ("... k's factors", dict(gk=at(9))), ("... q's factors", dict(gq=at(9))),
])
def test_kv_append(pkg, name, kw):
    L = pkg.lib()
    q, k, v = (pkg.Heads(kw.get(x, at(i + 1)), 512, 64) for i, x in enumerate("qkv"))
    qo = pkg.Heads(kw.get("qo", at(4)), kw.get("qo_row", 512), 64)
    c = cache_arg(pkg)
    rc = L.tsp_kv_append(ctypes.byref(c), ctypes.byref(k), ctypes.byref(v), 2, 100, vp(kw.get("off", at(5))), 2, vp(kw.get("table", at(6))), 7,
                         vp(kw.get("lengths", at(7))), ctypes.byref(q), 8, vp(kw.get("pos", at(8))), 3, (ctypes.c_int * 3)(10, 10, 10), 1e4, 0,
                         vp(kw.get("gq", at(10))), vp(kw.get("gk", at(11))), 1e-6, ctypes.byref(qo), NULL)
    assert rc == 1 and ("overlap no other tensor" in err(pkg) or "the cache overlaps" in err(pkg)), (name, rc, err(pkg))
