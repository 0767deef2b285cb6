"""CPU tests of the transformer pieces' limits: calls at the edge of what the kernels hold are refused with a
status and a message before any device work."""
from __future__ import annotations

import ctypes
import math

FAKE = ctypes.c_void_p(0x1000)   # never dereferenced


def test_attention_scale(pkg):
    """scale * log2(e), which the kernels multiply by, has to be finite as scale itself."""
    L = pkg.lib()
    q, k, v, o = (pkg.Heads(0x10000 * (i + 1), 512, 64) for i in range(4))
    for scale in (3.0e38, math.inf, math.nan, 0.0, -1.0):
        assert L.tsp_attention(q, k, v, 2, 100, 100, 8, 8, 64, FAKE, FAKE, 2, scale, 0, o, None, 0, None) == 1
        assert "scale" in L.tsp_last_error().decode()
