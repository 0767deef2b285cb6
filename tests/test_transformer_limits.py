"""CPU tests of the transformer pieces' limits: calls at the edge of what the kernels hold are refused with a
status and a message before any device work."""
from __future__ import annotations

import ctypes
import math
import types

import pytest

FAKE = ctypes.c_void_p(0x1000)   # never dereferenced


def test_attention_scale(pkg):
    """scale * log2(e), which the kernels multiply by, has to be finite as scale itself."""
    L = pkg.lib()
    q, k, v, o = (pkg.Heads(0x10000 * (i + 1), 512, 64) for i in range(4))
    for scale in (3.0e38, math.inf, math.nan, 0.0, -1.0):
        assert L.tsp_attention(q, k, v, 2, 100, 100, 8, 8, 64, FAKE, FAKE, 2, scale, 0, o, None, 0, None) == 1
        assert "scale" in L.tsp_last_error().decode()


def test_group_norm_partial_overlap(pkg):
    """An output that shares some of x's bytes but does not begin with them would be read after it is written."""
    L = pkg.lib()
    n, c = 100, 64
    for xd, od in ((0, 0), (0, 2), (1, 0), (2, 2)):
        size = {0: 4, 1: 2, 2: 2}
        xb, ob = n * c * size[xd], n * c * size[od]
        for x, out in ((0x100000, 0x100000 + xb - 16), (0x100000, 0x100000 + 16), (0x100000 + ob - 16, 0x100000), (0x100000 + c * 2, 0x100000)):
            rc = L.tsp_group_norm(ctypes.c_void_p(x), xd, n, c, 8, None, 1, None, None, 1e-6, 0, ctypes.c_void_p(out), od,
                                  ctypes.c_void_p(0x900000), 1 << 20, None)
            assert rc == 1 and "overlaps" in L.tsp_last_error().decode()


@pytest.mark.parametrize("private", [True, False])
def test_current_stream_without_the_private_call(pkg, monkeypatch, private):
    """The pieces' calls go to the current stream, by torch's public interface where the other one is not there."""
    import torch
    streams = []
    if private:
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    else:
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda i: types.SimpleNamespace(cuda_stream=100 + i))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    pkg._launch(torch.device("cuda", 3), None, lambda s, keep: streams.append(s))
    assert streams == [103]
