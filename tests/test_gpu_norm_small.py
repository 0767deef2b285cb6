"""GPU tests of norms whose mean square is below fp32's normal range: rows of zeros but for a few values, eps 0."""
from __future__ import annotations

import pytest

import served_ref as sr
import transformer_ref as ref
from test_gpu_served import check_mx, dtype, gen, ints

pytestmark = pytest.mark.gpu


def rows(n, c):
    """[n, c]: every 40th value some 2e-19, whose square (4e-38) is a normal number, and a mean square of some 1e-39, which is none: fp32
    holds it to 2^-21 of itself."""
    import torch
    x = torch.zeros((n, c), device="cuda")
    x[:, ::40] = 2e-19 * (1 + 0.2 * gen(c)(n, -(-c // 40))).clamp(0.6, 1.4)
    return x


@pytest.mark.parametrize("n,c", [(3, 512), (3, 1000), (4, 500), (5, 501), (2, 4096), (2, 1500), (2, 1501), (3, 8192), (2, 20_000), (2, 5001)])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(gpu_lib, n, c, residual):
    import torch
    print(f"[small rms norm] {n} x {c}", flush=True)
    x = rows(n, c)
    r = torch.zeros_like(x) if residual else None
    out = gpu_lib.rms_norm(x, eps=0.0, residual=r)
    y, _ = sr.rms_norm(x, r, None, 0.0)
    assert 1 < y.abs().max().item() < 30
    ref.check(out[0] if residual else out, y, y.abs() * sr.NORM_SLACK, "rms norm")
    if c % 32 == 0:
        check_mx(gpu_lib.rms_norm(x, eps=0.0, out_dtype=torch.float8_e4m3fn), y, "8 bits")


@pytest.mark.parametrize("held", ["mx4", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_append(gpu_lib, held, d):
    """The queries and the keys."""
    import torch
    n = 20
    cache = gpu_lib.kv_cache(2, 16, 2, d, "mx4" if held == "mx4" else dtype(held))
    table = ints([[1, 0]])
    q, k, v = rows(n * 4, d).view(n, 4, d), rows(n * 2, d).view(n, 2, d), gen(2)(n, 2, d)
    gq, gk = 1 + 0.2 * gen(3)(4, d), 1 + 0.2 * gen(4)(2, d)
    out = gpu_lib.kv_append(cache, k, v, table, ints([n]), q=q, q_gamma=gq, k_gamma=gk, eps=0.0)
    zero = torch.zeros((n, 1), dtype=torch.int32, device="cuda")
    yq, sq = ref.rope(q, zero, [0], 10000.0, True, gq, 0.0)
    yk, sk = ref.rope(k, zero, [0], 10000.0, True, gk, 0.0)
    assert 1 < yq.abs().max().item() < 30
    ref.check(out, yq, sq + yq.abs() * 2.0 ** -20, "q")
    kd = sr.keys_of(cache, table, [n], 0)[0]
    if held == "mx4":
        assert torch.equal(kd, sr.mx4_values(yk))
    else:
        ref.check(kd.to(dtype(held)), yk, sk + yk.abs() * 2.0 ** -20, "k")


@pytest.mark.parametrize("d", [64, 128])
def test_rope(gpu_lib, d):
    import torch
    n = 20
    q, gq = rows(n * 4, d).view(n, 4, d), 1 + 0.2 * gen(3)(4, d)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous()
    out = gpu_lib.rope_axes(q, pos, q_gamma=gq, eps=0.0)
    y, slack = ref.rope(q, pos, [d // 2], 10000.0, True, gq, 0.0)
    ref.check(out, y, slack + y.abs().amax(-1, keepdim=True) * 2.0 ** -20, "rope")
