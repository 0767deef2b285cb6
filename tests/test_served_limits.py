"""CPU tests of the cached attention's limits: sizes past them are refused before any device work, and need no workspace that
a caller would allocate for nothing."""
from __future__ import annotations

import ctypes

import pytest

MOST = (1 << 31) - 1


@pytest.mark.parametrize("nq,samples,hq,heads,max_pages,page", [
    (MOST, 1, 4096, 1, 7, 16),            # rows
    (100, 2, 8192, 8, 7, 16),             # heads
    (100, 2, 8, 8, 1 << 28, 16),          # keys
    (100, 2, 8, 8, MOST, 256),
    (1 << 28, 1, 4096, 4096, 1000, 16),   # units of rows and heads: 2^33
    (100, MOST, 4096, 4096, 1000, 16),
    (MOST, MOST, 4096, 4096, MOST, 256),
])
def test_past_the_limits(pkg, nq, samples, hq, heads, max_pages, page):
    L = pkg.lib()
    c = pkg.KvCacheArg(9 << 32, 100, page, heads, 64, pkg.TSP_KV_MX4)
    assert L.tsp_attention_cached_workspace_bytes(nq, samples, hq, ctypes.byref(c), max_pages) == 0
    q, o = pkg.Heads(1 << 50, hq * 64, 64), pkg.Heads(1 << 55, hq * 64, 64)
    rc = L.tsp_attention_cached(ctypes.byref(q), 2, nq, hq, ctypes.byref(c), ctypes.c_void_p(5 << 32), samples, ctypes.c_void_p(1 << 60),
                                max_pages, ctypes.c_void_p(7 << 32), 0.125, 1, ctypes.byref(o), ctypes.c_void_p(8 << 32), 1 << 40, None)
    assert rc == 1, rc


def test_within_them(pkg):
    """Sizes at the limits have a workspace of some size: at most 768 workgroups' pieces of 32 rows, or 512 of 256."""
    L = pkg.lib()
    for nq, samples, hq, heads, max_pages in ((1, 1, 8, 8, ((1 << 31) - (1 << 16) - 1) // 16), ((1 << 31) - 2048, 1, 1, 1, 1000), (1 << 16, 1 << 16, 4096, 4096, 10)):
        c = pkg.KvCacheArg(9 << 32, 100, 16, heads, 128, pkg.TSP_KV_MX4)
        need = L.tsp_attention_cached_workspace_bytes(nq, samples, hq, ctypes.byref(c), max_pages)
        assert 0 < need <= 512 * (256 * (128 * 4 + 8) + 16)
