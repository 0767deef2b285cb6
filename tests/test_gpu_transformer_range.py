"""GPU tests of attention at the ends of its number range: keys that weigh little each and something together,
scores far from zero, against their 64-bit forms; of group norm's factors off a 16-byte boundary; and of captured
calls replayed with other lengths."""
from __future__ import annotations

import math

import pytest

import transformer_ref as ref

pytestmark = pytest.mark.gpu


def dtype(key):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[key]


@pytest.mark.parametrize("key,gap,lk,d,at", [("f16", 17.0, 200_000, 64, 0), ("f16", 17.4, 200_000, 128, 0), ("f16", 17.4, 200_000, 64, 70),
                                             ("f16", 15.0, 600_000, 64, 0), ("f16", 17.4, 100_001, 32, 33), ("f16", 20.0, 600_000, 64, 1),
                                             ("bf16", 17.4, 2_400_000, 64, 0), ("bf16", 17.4, 2_400_001, 128, 70), ("f32", 17.4, 30_000, 64, 0)])
@pytest.mark.parametrize("rows", [100_000, 3])
def test_attention_keys_far_below_the_largest(gpu_lib, key, gap, lk, d, at, rows):
    """One key `gap` nats above all others, its value 0 and theirs 1: the output is the others' weight, which
    rounding must not take or add. Enough rows for the keys not to be split, and few."""
    import torch
    if key == "f32" and rows > 3:
        rows = 40_000
    print(f"[far below] {key} gap={gap} lk={lk} d={d} rows={rows}", flush=True)
    q, k = torch.zeros(1, 1, d, device="cuda"), torch.zeros(lk, 1, d, device="cuda")
    q[..., 0] = 4.0
    k[at, 0, 0] = gap / 4.0
    v = torch.ones(lk, 1, d, device="cuda", dtype=dtype(key))
    v[at] = 0
    q, k = q.to(dtype(key)), k.to(dtype(key))
    out = gpu_lib.attention(q.expand(rows, 1, d).contiguous(), k, v, scale=1.0)
    s = (k.double()[:, 0] @ q.double()[0, 0])
    p = torch.softmax(s, dim=0)
    small = 1 - p[at].item()
    # Of the others' weight: half a step of p in the 16-bit type, 2^-12 for the score and the exponent, and their
    # sum, a matrix core's over 16 keys (fp32: 2) at a time, by half a step of what is summed so far an addition, so of
    # half the sum in the mean. Of all weight, which is divided by: the tiles of 64 (fp32: 32) keys added and a tile's 16
    # additions. f16 below its normal range, 2^-25 of the largest and kept 2^-11 lower: 2^-36 a key.
    half, keys, tile = (0.0, 2, 32) if key == "f32" else (ref.half_step(dtype(key)), 16, 64)
    bound = small * (half + 2.0 ** -12 + (lk / keys / 2 + lk / tile + 16) * 2.0 ** -24)
    if key == "f16":
        bound += lk * 2.0 ** -36
    bound += ref.half_step(dtype(key)) * (small + bound) + (2.0 ** -25 if key == "f16" else 0.0)
    assert small > 2 * bound       # all of it lost would show
    worst = (out.double() - small).abs().max().item()
    print(f"  others weigh {small:.6f}, off by {worst:.3g}, bound {bound:.3g}", flush=True)
    assert worst <= bound


@pytest.mark.parametrize("e", [12, 18, 24, 28, 33])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("key", ["f16", "bf16", "f32"])
def test_attention_scores_far_from_zero(gpu_lib, e, sign, order, key):
    """Scores of +-2^e with a few units between them, all of them exact in fp32: only differences count, whatever the
    units are worth. (The largest score by itself, times scale * log2(e) in fp32, is up to 2^10 off.)"""
    import torch
    print(f"[far scores] 2^{e} {sign} {order} {key}", flush=True)
    unit = 1 << max(0, e - 22)       # of a score: 24 bits below 2^(e + 1)
    a = (e - 2) // 2
    g = torch.Generator(device="cuda")
    g.manual_seed(e)
    for rows, lk, d, causal in ((1, 20_000, 128, False), (200, 1000, 64, True), (300, 700, 32, False)):
        j = torch.arange(lk, device="cuda") * 255 // (lk - 1)
        if order == "falling":
            j = j.flip(0)
        elif order == "mixed":
            j = j[torch.randperm(lk, device="cuda", generator=g)]
        q, k = torch.zeros(rows, 1, d, device="cuda"), torch.zeros(lk, 1, d, device="cuda")
        q[..., :8], k[..., :8] = 2.0 ** a, sign * 2.0 ** (e - 3 - a)
        q[..., 8], k[:, 0, 8] = float(unit), j.float()
        v = torch.randn(lk, 1, d, device="cuda", generator=g)
        q, k, v = q.to(dtype(key)), k.to(dtype(key)), v.to(dtype(key))
        for scale in (1.0, 0.375 / unit):
            out = gpu_lib.attention(q, k, v, causal=causal, scale=scale)
            o, slack = ref.attention(q, k, v, [0, rows], [0, lk], causal, scale)
            ref.check(out, o, slack, f"{rows} rows, scale {scale:.3g}")


@pytest.mark.parametrize("n,c,groups", [(700, 64, 8), (60_000, 256, 32)])
def test_group_norm_factors_inside_a_buffer(gpu_lib, n, c, groups):
    """gamma and beta as slices of one parameter buffer, off a 16-byte boundary: the same kernels, so the same bits."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    x, f = torch.randn(n, c, device="cuda", generator=g), torch.randn(2 * c + 1, device="cuda", generator=g)
    gamma, beta = f[1:c + 1], f[c + 1:]
    assert gamma.data_ptr() % 16 and beta.data_ptr() % 16
    want = gpu_lib.group_norm(x, groups, gamma.clone(), beta.clone(), silu=True)
    for a, b in ((gamma, beta), (gamma.clone(), beta), (gamma, beta.clone())):
        assert torch.equal(gpu_lib.group_norm(x, groups, a, b, silu=True), want)


@pytest.mark.parametrize("rows", [1, 40])
def test_replayed_with_other_lengths(gpu_lib, rows):
    """A captured step replayed with other offsets in the same buffers, even and skewed: lengths are read on the
    device, so each replay gives what an eager call does, and rows outside the samples stay."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    samples, n = 16, 30_000
    nq = rows * samples
    q, k, v = (torch.randn(m, h, 64, device="cuda", generator=g).bfloat16() for m, h in ((nq, 4), (n, 2), (n, 2)))
    x = torch.randn(n, 64, device="cuda", generator=g)
    qo = torch.arange(0, nq + 1, rows, device="cuda", dtype=torch.int32)
    ko = torch.arange(0, n + 1, n // samples, device="cuda", dtype=torch.int32)[:samples + 1].contiguous()
    o, y = torch.empty_like(q), torch.empty_like(x)
    ws, wn = gpu_lib.attention_workspace(nq, n, samples, 4, 2, 64), gpu_lib.group_norm_workspace(n, 64, 8, samples)

    def call():
        gpu_lib.attention(q, k, v, qo, ko, causal=True, out=o, workspace=ws)
        gpu_lib.group_norm(x, 8, silu=True, offsets=ko, out=y, workspace=wn)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lengths in ([1800] * 16, [10] * 5 + [29_000] + [0] * 10, [100 * i for i in range(16)], [n // 16] * 16):
        bounds = ref.offsets_of(lengths)
        ko.copy_(torch.tensor(bounds, dtype=torch.int32))
        o.fill_(-7), y.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone(), y.clone()
        o.fill_(-7), y.fill_(-7)
        call()
        torch.cuda.synchronize()
        assert torch.equal(got[0], o) and torch.equal(got[1], y) and (y[bounds[-1]:] == -7).all()
        want, slack = ref.attention(q, k, v, ref.offsets_of([rows] * samples), bounds, True, 0.125)
        ref.check(o, want, slack, "replay")
