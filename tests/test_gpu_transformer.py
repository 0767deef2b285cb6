"""GPU tests of the transformer pieces over packed rows: group_norm, rope_axes and attention against
their 64-bit forms, at the sizes, masks, strides and values where they can go wrong; streams, captured
graphs, and a block of them run together."""
from __future__ import annotations

import math

import pytest

import transformer_ref as ref

pytestmark = pytest.mark.gpu

KEYS = ["f32", "f16", "bf16"]


def dtype(key):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[key]


def gen(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *shape: torch.randn(shape, generator=g, device="cuda")


def ints(values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- group norm ---------------------------------------------------------------------------------
GN_CASES = [
    # lengths, c, groups
    ([1], 8, 1), ([1], 64, 32), ([2], 7, 7), ([15], 30, 5), ([17], 64, 64), ([300], 96, 32), ([33, 0, 1, 260], 64, 8),
    ([0, 0, 5], 40, 4), ([2606], 64, 32), ([513, 4, 1030], 320, 32), ([90], 4096, 32), ([31], 4104, 8), ([3], 5000, 1000),
    ([1] * 130 + [70], 32, 8), ([40_000, 3], 128, 32), ([1025], 1024, 16), ([12_345], 20, 5), ([700, 1], 1536, 3),
]


@pytest.mark.parametrize("case", range(len(GN_CASES)))
@pytest.mark.parametrize("xk,ok", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16")])
def test_group_norm(gpu_lib, case, xk, ok):
    lengths, c, groups = GN_CASES[case]
    n = sum(lengths)
    print(f"[group norm] {lengths[:6]} c={c} groups={groups} {xk}->{ok}", flush=True)
    randn = gen(case)
    x = (randn(n, c) * (0.2 + randn(c).abs()) + randn(c)).to(dtype(xk))
    gamma, beta = (None, None) if case % 3 == 0 else (1 + 0.3 * randn(c), 0.3 * randn(c))
    bounds = ref.offsets_of(lengths)
    silu = case % 2 == 0
    out = gpu_lib.group_norm(x, groups, gamma, beta, eps=1e-5, silu=silu, offsets=ints(bounds), out_dtype=dtype(ok))
    assert out.dtype == dtype(ok)
    y, slack = ref.group_norm(x, groups, bounds, gamma, beta, 1e-5, silu)
    ref.check(out, y, slack, "group norm")
    if len(lengths) == 1:
        import torch
        assert torch.equal(out, gpu_lib.group_norm(x, groups, gamma, beta, eps=1e-5, silu=silu, out_dtype=dtype(ok)))


@pytest.mark.parametrize("c,groups", [(64, 8), (60, 4)])
def test_group_norm_far_mean_and_constant(gpu_lib, c, groups):
    """A mean a thousand times the spread, and a group of equal values (variance 0)."""
    randn = gen(5)
    x = randn(4001, c) + 1000.0
    x[:, : c // groups] = 3.25
    y, slack = ref.group_norm(x, groups, [0, 4001], None, None, 1e-6, False)
    out = gpu_lib.group_norm(x, groups, eps=1e-6)
    ref.check(out, y, slack, "far mean")
    assert (out[:, : c // groups] == 0).all()


@pytest.mark.parametrize("n,c,groups,bounds", [(4096, 64, 32, None), (2049, 64, 8, [0, 1024, 1025, 1025, 2049]), (3001, 24, 24, [5, 3000]),
                                               (1100, 64, 4, None), (9000, 64, 32, None), (500, 60, 4, None)])
def test_group_norm_in_place(gpu_lib, n, c, groups, bounds):
    """In place and apart, the same values."""
    import torch
    randn = gen(n)
    x, gamma = randn(n, c), randn(c)
    off = None if bounds is None else ints(bounds)
    y, slack = ref.group_norm(x, groups, bounds or [0, n], gamma, None, 1e-6, True)
    lo, hi = (0, n) if bounds is None else (bounds[0], bounds[-1])
    out = gpu_lib.group_norm(x, groups, gamma, silu=True, offsets=off)
    ref.check(out[lo:hi], y[lo:hi], slack[lo:hi], "apart")
    assert gpu_lib.group_norm(x, groups, gamma, silu=True, offsets=off, out=x) is x and torch.equal(x[lo:hi], out[lo:hi])


@pytest.mark.parametrize("n,c,groups", [(900, 64, 8), (900, 64, 32), (30_000, 64, 8), (30_000, 8, 1), (9000, 64, 32), (9000, 128, 64), (60_000, 36, 4), (40, 4104, 8)])
@pytest.mark.parametrize("rows", [1, 40, 400])
def test_group_norm_outliers_first(gpu_lib, n, c, groups, rows):
    """The first row, or the first few, far from all others: the sums must not go about its values (a variance of
    n values is then one n-th of what is summed)."""
    randn = gen(rows)
    x = randn(n, c)
    x[:min(rows, n // 2)] += 3.0e4
    y, slack = ref.group_norm(x, groups, [0, n], None, None, 1e-6, False)
    ref.check(gpu_lib.group_norm(x, groups), y, slack, "outliers first")


@pytest.mark.parametrize("c,groups", [(64, 8), (36, 4)])
def test_group_norm_leaves_other_rows(gpu_lib, c, groups):
    """Rows before the first and behind the last sample keep what out held; a NaN stays in its sample and
    group; in place; a workspace full of NaN."""
    import torch
    randn = gen(6)
    x = randn(500, c)
    bounds = [7, 107, 107, 400]
    x[50, 3] = math.nan
    x[450] = math.inf
    out = torch.full((500, c), -7.0, device="cuda")
    ws = gpu_lib.group_norm_workspace(500, c, groups, 3)
    ws.fill_(255)
    gpu_lib.group_norm(x, groups, offsets=ints(bounds), out=out, workspace=ws)
    assert (out[:7] == -7).all() and (out[400:] == -7).all()
    y, slack = ref.group_norm(x, groups, bounds, None, None, 1e-6, False)
    ref.check(out[7:400], y[7:400], slack[7:400], "rows")
    assert torch.isnan(out[7:107, : c // groups]).all() and torch.isfinite(out[7:107, c // groups:]).all()
    z = x.clone()
    assert gpu_lib.group_norm(z, groups, offsets=ints(bounds), out=z) is z
    assert torch.equal(z[7:400].nan_to_num(9), out[7:400].nan_to_num(9)) and torch.equal(z[:7], x[:7])


def test_group_norm_silu_far(gpu_lib):
    """silu of +-100 and beyond: no NaN from an exp that overflows."""
    import torch
    x = torch.tensor([[-1.0, 1.0]], device="cuda").repeat(64, 4)
    beta = torch.tensor([200.0, -200.0] * 4, device="cuda")
    gamma = torch.full((8,), 50.0, device="cuda")
    y, slack = ref.group_norm(x, 2, [0, 64], gamma, beta, 1e-6, True)
    ref.check(gpu_lib.group_norm(x, 2, gamma, beta, silu=True), y, slack, "silu")


def test_group_norm_unaligned(gpu_lib):
    import torch
    randn = gen(8)
    buf = randn(1 + 300 * 64).half()
    x = buf[1:].reshape(300, 64)
    y, slack = ref.group_norm(x, 8, [0, 300], None, None, 1e-6, False)
    ref.check(gpu_lib.group_norm(x, 8), y, slack, "unaligned")
    ref.check(gpu_lib.group_norm(x.t().contiguous().t(), 8), y, slack, "transposed")
    assert gpu_lib.group_norm(x[:0], 8).shape == (0, 64)


def test_group_norm_unaligned_factors(gpu_lib):
    randn = gen(18)
    x, f = randn(700, 64), randn(129)
    for gamma, beta in ((f[1:65], None), (None, f[65:]), (f[1:65], f[65:])):
        y, slack = ref.group_norm(x, 8, [0, 700], gamma, beta, 1e-6, True)
        ref.check(gpu_lib.group_norm(x, 8, gamma, beta, silu=True), y, slack, "factors")


def test_group_norm_bad_offsets_stay_inside(gpu_lib):
    """Offsets out of order or outside [0, n]: no row outside the tensor is read or written."""
    import torch
    randn = gen(9)
    x = randn(400, 64)
    for bounds in ([-50, 100, 9000], [300, 20, 400], [2**31 - 1, 5, 7], [0, 2**31 - 1, -2**31]):
        guard = torch.full((600, 64), -7.0, device="cuda")
        gpu_lib.group_norm(x, 8, offsets=ints(bounds), out=guard[100:500])
        assert (guard[:100] == -7).all() and (guard[500:] == -7).all()


@pytest.mark.parametrize("n,c", [(6000, 64), (20_000, 64), (6000, 60), (20_000, 60)])
def test_group_norm_bad_offsets_in_the_workspace(gpu_lib, n, c):
    """Offsets that name the same rows again and again have more units than the workspace holds: nothing behind
    it is read (there are NaN there) or written."""
    import torch
    x = gen(19)(n, c)
    need = gpu_lib.group_norm_workspace(n, c, 4, 5).numel()
    ws = torch.full((16 * need,), 255, dtype=torch.uint8, device="cuda")
    guard = torch.full((n + 200, c), -7.0, device="cuda")
    gpu_lib.group_norm(x, 4, offsets=ints([0, n, 0, n, 0, n]), out=guard[100:100 + n], workspace=ws[:need])
    assert (guard[:100] == -7).all() and (guard[100 + n:] == -7).all() and (ws[need:] == 255).all()
    assert torch.isfinite(guard).all() and (guard[100:100 + n] != -7).all()


# ---- rotary positions ---------------------------------------------------------------------------
ROPE_CASES = [
    # n, hq, hk, d, pairs, interleaved
    (1, 1, 0, 8, [4], True), (1, 1, 1, 8, [1, 1, 1, 1], False), (97, 16, 16, 64, [16, 16], False), (33, 3, 1, 128, [21, 21, 21], True),
    (40, 5, 2, 80, [13, 13, 13], False), (257, 8, 8, 96, [16, 0, 30], True), (19, 2, 2, 256, [128], False), (21, 4, 4, 40, [5], True),
    (1000, 12, 12, 32, [8, 8], True), (37, 2, 1, 256, [40, 40, 40], True), (65, 1, 2, 200, [33, 33, 33], False), (3, 40, 8, 24, [0, 12], False), (5, 1, 7, 104, [30, 20], True), (2048, 16, 4, 64, [10, 10, 10], True),
]


@pytest.mark.parametrize("case", range(len(ROPE_CASES)))
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("xk,ok", [("f32", "f32"), ("bf16", "bf16"), ("f32", "f16"), ("f16", "f16")])
def test_rope(gpu_lib, case, norm, xk, ok):
    import torch
    n, hq, hk, d, pairs, inter = ROPE_CASES[case]
    print(f"[rope] {ROPE_CASES[case]} norm={norm} {xk}->{ok}", flush=True)
    randn = gen(case)
    q, k = randn(n, hq, d).to(dtype(xk)), randn(n, hk, d).to(dtype(xk)) if hk else None
    far = [100, 1 << 21, 1 << 27][case % 3]
    pos = torch.randint(-far, far, (n, len(pairs)), device="cuda", dtype=torch.int32)
    gq, gk = (1 + 0.3 * randn(hq, d), 1 + 0.3 * randn(hk, d) if hk else None) if norm else (None, None)
    got = gpu_lib.rope_axes(q, pos, k=k, pairs=pairs, interleaved=inter, q_gamma=gq, k_gamma=gk, eps=1e-5, out_dtype=dtype(ok))
    for x, o, g, name in ((q, got[0] if hk else got, gq, "q"), (k, got[1] if hk else None, gk, "k")):
        if x is None:
            continue
        y, slack = ref.rope(x, pos, pairs, 10000.0, inter, g, 1e-5)
        ref.check(o, y, slack, name)


def test_rope_views_in_place(gpu_lib):
    """q and k as views into one linear's output, turned where they lie; v and the rest stay."""
    import torch
    randn = gen(3)
    qkv = randn(101, 3, 8, 64).bfloat16()
    before = qkv.clone()
    pos = torch.randint(0, 64, (101, 3), device="cuda", dtype=torch.int32)
    q, k = qkv[:, 0], qkv[:, 1]
    rq, rk = gpu_lib.rope_axes(q, pos, k=k, q_out=q, k_out=k)
    assert rq.data_ptr() == qkv.data_ptr() and torch.equal(qkv[:, 2], before[:, 2])
    for o, x in ((rq, before[:, 0]), (rk, before[:, 1])):
        y, slack = ref.rope(x, pos, [10, 10, 10], 10000.0, True, None, 0)
        ref.check(o, y, slack, "in place")
    # heads first, and a view that starts off a 16-byte boundary (copied)
    hm = randn(8, 101, 64).half().transpose(0, 1)
    y, slack = ref.rope(hm, pos, [10, 10, 10], 10000.0, True, None, 0)
    ref.check(gpu_lib.rope_axes(hm, pos), y, slack, "heads first")
    odd = randn(101 * 8 * 64 + 3).half()[3:].reshape(101, 8, 64)
    y, slack = ref.rope(odd, pos, [10, 10, 10], 10000.0, True, None, 0)
    ref.check(gpu_lib.rope_axes(odd, pos), y, slack, "unaligned")
    dst = torch.full((8, 101, 72), -7.0, device="cuda", dtype=torch.float16)
    gpu_lib.rope_axes(odd, pos, q_out=dst[:, :, :64].transpose(0, 1))
    ref.check(dst[:, :, :64].transpose(0, 1), y, slack, "out heads first")
    assert (dst[:, :, 64:] == -7).all()


def test_rope_unaligned_gamma(gpu_lib):
    import torch
    randn = gen(7)
    x, pos = randn(50, 2, 64), torch.randint(0, 64, (50, 3), device="cuda", dtype=torch.int32)
    g = randn(2 * 64 + 1)[1:].view(2, 64)
    y, slack = ref.rope(x, pos, [10, 10, 10], 10000.0, True, g, 1e-6)
    ref.check(gpu_lib.rope_axes(x, pos, q_gamma=g), y, slack, "gamma")
    y, slack = ref.rope(x[:1].expand(50, 2, 64), pos, [10, 10, 10], 10000.0, True, None, 1e-6)
    ref.check(gpu_lib.rope_axes(x[:1].expand(50, 2, 64), pos), y, slack, "broadcast row")


def test_rope_values(gpu_lib):
    """A zero row stays zero under the norm; an Inf or a NaN stays in its pair (its head with the norm);
    position 0 changes nothing; no rows."""
    import torch
    randn = gen(4)
    x = randn(10, 2, 64)
    x[3] = 0
    x[4, 1, 6] = math.nan
    pos = torch.arange(10, device="cuda", dtype=torch.int32)[:, None] * 1000
    y = gpu_lib.rope_axes(x, pos)
    assert torch.equal(y[0], x[0]) and (y[3] == 0).all()
    bad = torch.isnan(y[4, 1]).nonzero().flatten().tolist()
    assert bad == [6, 7] and torch.isfinite(y[4, 0]).all()
    z = gpu_lib.rope_axes(x, pos, q_gamma=torch.ones(2, 64, device="cuda"), eps=1e-6)
    assert (z[3] == 0).all() and torch.isnan(z[4, 1]).all() and torch.isfinite(z[4, 0]).all()
    assert gpu_lib.rope_axes(x[:0], pos[:0]).shape == (0, 2, 64)


# ---- attention ----------------------------------------------------------------------------------
AT_CASES = [
    # (q length, k length) of each sample, hq, hkv, d
    ([(1, 1)], 1, 1, 8), ([(1, 63)], 4, 2, 64), ([(1, 64)], 1, 1, 128), ([(2, 65)], 8, 1, 40), ([(33, 129)], 2, 2, 64),
    ([(64, 64)], 3, 3, 128), ([(130, 257)], 4, 4, 80), ([(257, 130)], 4, 2, 96), ([(5, 0), (0, 7), (64, 64), (130, 257)], 4, 2, 64),
    ([(0, 0), (1, 1), (0, 0), (31, 32), (32, 31)], 6, 3, 128), ([(1, 1)] * 70 + [(40, 200)], 2, 1, 32), ([(1000, 1000)], 2, 1, 128),
    ([(511, 513), (300, 299), (3, 700)], 8, 2, 64), ([(129, 640)], 5, 5, 16), ([(70, 300)], 16, 1, 128), ([(1, 5000)], 16, 2, 128),
    ([(3, 9001), (1, 64), (8, 2)], 8, 8, 64), ([(2606, 2606)], 2, 2, 64), ([(40, 20_011)], 2, 1, 72), ([(700, 1029)], 4, 4, 64),
]


@pytest.mark.parametrize("case", range(len(AT_CASES)))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("key", ["f16", "bf16", "f32"])
def test_attention(gpu_lib, case, causal, key):
    lens, hq, hkv, d = AT_CASES[case]
    print(f"[attention] {lens[:6]} heads {hq}/{hkv} d={d} causal={causal} {key}", flush=True)
    import torch
    randn = gen(case)
    qb, kb = ref.offsets_of([a for a, _ in lens]), ref.offsets_of([b for _, b in lens])
    q, k, v = (randn(m, h, d).to(dtype(key)) for m, h in ((qb[-1], hq), (kb[-1], hkv), (kb[-1], hkv)))
    out = gpu_lib.attention(q, k, v, ints(qb), ints(kb), causal=causal)
    o, slack = ref.attention(q, k, v, qb, kb, causal, d ** -0.5)
    ref.check(out, o, slack, "attention")
    assert torch.equal(out, gpu_lib.attention(q, k, v, ints(qb), ints(kb), causal=causal))
    if len(lens) == 1:
        assert torch.equal(out, gpu_lib.attention(q, k, v, causal=causal))


@pytest.mark.parametrize("spread", [0.05, 6.0, 60.0])
@pytest.mark.parametrize("key", ["f16", "bf16"])
def test_attention_spread_and_growing_maximum(gpu_lib, spread, key):
    """Scores from flat to one-hot, and keys sorted so that every tile raises the maximum."""
    randn = gen(11)
    q, k, v = randn(150, 2, 64), randn(900, 2, 64), randn(900, 2, 64).to(dtype(key))
    import torch
    order = (k[:, 0] @ q[0, 0]).argsort()
    q, k = (q * spread).to(dtype(key)), k[order].to(dtype(key))
    out = gpu_lib.attention(q, k, v, scale=0.3)
    o, slack = ref.attention(q, k, v, [0, 150], [0, 900], False, 0.3)
    # a score of size s has fp32 rounding of about 64 s 2^-24 in its exponent
    top = (0.3 * (q.double().abs().amax() * k.double().abs().amax() * 64)).item()
    slack = slack * (1 + top * 64 * 2.0 ** -24 / 2.0 ** -12)
    ref.check(out, o, slack, f"spread {spread}")
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("key", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,lk", [(200, 20_000), (1, 20_000), (64, 130)])
@pytest.mark.parametrize("gap", [9.0, 10.5, 15.0])
def test_attention_many_small_probabilities(gpu_lib, key, rows, lk, gap):
    """One key far above thousands of equal ones, whose probabilities are below f16's normal range and together
    weigh as much as its: they count in the sums as in the products."""
    import torch
    d = 64
    q = torch.zeros(rows, 1, d, device="cuda")
    q[:, 0, 0] = 4.0
    k = torch.zeros(lk, 1, d, device="cuda")
    k[lk // 2, 0, 0] = gap / 4.0
    randn = gen(lk)
    q, k, v = q.to(dtype(key)), k.to(dtype(key)), (randn(lk, 1, d) * 0.1 + 1.0).to(dtype(key))
    out = gpu_lib.attention(q, k, v, scale=1.0)
    s = (q.double()[:, 0] @ k.double()[:, 0].t())
    p = torch.softmax(s, dim=1)
    want = (p @ v.double()[:, 0])[:, None]
    # f16: a probability of 2^-24 units is off by half a unit, in the sum and in the product alike
    rel = {"f16": 2.0 ** -11 + 2.0 ** -25 * math.exp(gap), "bf16": 2.0 ** -8, "f32": 2.0 ** -20 + lk * 2.0 ** -25}[key]
    slack = torch.full_like(want, 2 * rel + 2.0 ** -12 + lk * 2.0 ** -25) * v.double().abs().max()
    ref.check(out, want, slack, "small probabilities")


def test_attention_views(gpu_lib):
    """Views into one linear's output, heads first, unaligned, a head shared by broadcasting, and an output
    that is a view with other columns in it."""
    import torch
    randn = gen(12)
    qkv = randn(333, 3, 4, 64).half()
    q, k, v = qkv.unbind(1)
    o, slack = ref.attention(q, k, v, [0, 333], [0, 333], True, 0.125)
    ref.check(gpu_lib.attention(q, k, v, causal=True), o, slack, "fused")
    hm = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (q, k, v)]
    ref.check(gpu_lib.attention(*hm, causal=True), o, slack, "heads first")
    off = [torch.cat([t.new_zeros(1), t.flatten()])[1:].reshape(333, 4, 64) for t in (q, k, v)]
    ref.check(gpu_lib.attention(*off, causal=True), o, slack, "unaligned")
    dst = torch.full((333, 4, 96), -7.0, device="cuda", dtype=torch.float16)
    gpu_lib.attention(q, k, v, causal=True, out=dst[:, :, 16:80])
    ref.check(dst[:, :, 16:80], o, slack, "out view")
    assert (dst[:, :, :16] == -7).all() and (dst[:, :, 80:] == -7).all()
    one = k[:, :1].expand(333, 4, 64)
    o, slack = ref.attention(q, one, v, [0, 333], [0, 333], False, 0.125)
    ref.check(gpu_lib.attention(q, one, v), o, slack, "broadcast head")
    same = v[:1].expand(333, 4, 64)
    out = gpu_lib.attention(q, k, same)
    assert ((out - same).abs() <= 2.0 ** -9 * same.abs()).all()      # a mean of equal rows, p rounded to half steps


@pytest.mark.parametrize("d", [8, 24, 32, 40, 56, 72, 80, 88, 96, 104, 120])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("key", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("lq,lk,hq,hkv", [(300, 1000, 2, 1), (5, 3001, 4, 2), (129, 64, 1, 1)])
def test_attention_widths(gpu_lib, d, causal, key, lq, lk, hq, hkv):
    """Heads of widths that are none of the kernels' own, as views beside other values and into an output whose
    other columns stay."""
    import torch
    randn = gen(d)
    q, kv = randn(lq, hq, d + 8).to(dtype(key)), randn(lk, 2, hkv, d + 16).to(dtype(key))
    q[:, :, d:], kv[..., d:] = math.nan, math.inf
    q, k, v = q[:, :, :d], kv[:, 0, :, :d], kv[:, 1, :, :d]
    out = torch.full((lq, hq, d + 8), -7.0, device="cuda", dtype=dtype(key))
    gpu_lib.attention(q, k, v, causal=causal, out=out[:, :, 8:])
    o, slack = ref.attention(q, k, v, [0, lq], [0, lk], causal, d ** -0.5)
    ref.check(out[:, :, 8:], o, slack, f"width {d}")
    assert (out[:, :, :8] == -7).all()


@pytest.mark.parametrize("d", [64, 128, 40, 96, 32, 80])
@pytest.mark.parametrize("key", ["f16", "bf16", "f32"])
def test_attention_values_behind_the_mask(gpu_lib, d, key):
    """Infinities and NaN in keys and values that a row does not see: the next sample's, the rows between
    the samples, later keys of a causal sample. Rows that do see them get what the formula gives."""
    import torch
    randn = gen(13)
    qb, kb = [3, 73, 100], [10, 90, 150]
    q, k, v = (randn(m, 2, d).to(dtype(key)) for m in (110, 160, 160))
    k[:10], v[:10], k[150:], v[150:] = math.nan, math.inf, math.inf, math.nan
    k[90:] = math.nan            # the second sample's: the first sees none of it
    v[90:] = math.inf
    out = gpu_lib.attention(q, k, v, ints(qb), ints(kb))
    o, slack = ref.attention(q[3:73], k[10:90], v[10:90], [0, 70], [0, 80], False, d ** -0.5)
    ref.check(out[3:73], o, slack, "other sample")
    assert torch.isnan(out[73:100]).all()
    # causal: row i of 70 sees keys up to i + 10
    k, v = randn(160, 2, d).to(dtype(key)), randn(160, 2, d).to(dtype(key))
    k[70, 0], v[60, 1, 3], v[60, 0, 5], v[75, 1], v[33, 0, d - 1] = math.nan, math.inf, -math.inf, math.nan, math.nan
    out = gpu_lib.attention(q, k, v, ints(qb), ints(kb), causal=True)
    o, slack = ref.attention(q[3:73], k[10:90], v[10:90], [0, 70], [0, 80], True, d ** -0.5)
    ref.check(out[3:73], o, slack, "later keys")


@pytest.mark.parametrize("hkv,lq,lk", [(1, 4, 300), (2, 7, 20_000), (4, 3, 61), (1, 8, 7), (2, 40, 5000)])
@pytest.mark.parametrize("key", ["bf16", "f32"])
def test_attention_few_rows_behind_the_mask(gpu_lib, hkv, lq, lk, key):
    """The same for a few new tokens against a cache, split or not: the last keys hold an Inf and a NaN that
    the earlier tokens do not see."""
    import torch
    randn = gen(lk)
    q, k, v = (randn(m, h, 64).to(dtype(key)) for m, h in ((lq, 4), (lk, hkv), (lk, hkv)))
    k[-1, 0, 5], v[-2, hkv - 1, 63], v[-1, 0, 0] = math.inf, math.nan, -math.inf
    out = gpu_lib.attention(q, k, v, causal=True)
    o, slack = ref.attention(q, k, v, [0, lq], [0, lk], True, 0.125)
    ref.check(out, o, slack, "few rows")
    seen = max(0, lk - 2 - (lk - lq))
    assert torch.isfinite(out[:seen]).all()


SKEWED = [
    # query and key lengths: one long sample among short ones, few rows each or not
    ([1] * 16, [100] * 9 + [30_000] + [7] * 6), ([1] * 64, [20_000] + [65] * 63), ([3, 0, 8, 1, 2], [9000, 50, 0, 1, 3]),
    ([1, 1], [12_000, 1]), ([2] * 20, [64 * (i % 5) for i in range(19)] + [15_000]), ([300, 10, 1], [300, 6000, 40_000]),
    ([1] * 5, [5000] * 5), ([8] * 16, [5000 + 300 * i for i in range(16)]), ([33, 40, 5, 1], [33, 20_000, 70, 1]),
    ([0] * 7 + [1], [100] * 7 + [25_000]), ([1] * 65, [40_000] + [10] * 64),
]


@pytest.mark.parametrize("case", range(len(SKEWED)))
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (2, 2, 128), (12, 3, 96)])
@pytest.mark.parametrize("causal,key", [(True, "bf16"), (False, "f16"), (True, "f32")])
def test_attention_skewed_lengths(gpu_lib, case, hq, hkv, d, causal, key):
    """Splits by the samples' lengths: every row once, the same values again, rows behind the samples left."""
    import torch
    lq, lk = SKEWED[case]
    qb, kb = ref.offsets_of(lq), ref.offsets_of(lk)
    randn = gen(case)
    q, k, v = randn(qb[-1] + 2, hq, d).to(dtype(key)), randn(kb[-1] + 3, hkv, d).to(dtype(key)), randn(kb[-1] + 3, hkv, d).to(dtype(key))
    k[kb[-1]:], v[kb[-1]:] = math.nan, math.inf
    out = torch.full_like(q, -7.0)
    gpu_lib.attention(q, k, v, ints(qb), ints(kb), causal=causal, out=out)
    assert (out[qb[-1]:] == -7).all()
    o, slack = ref.attention(q, k, v, qb, kb, causal, d ** -0.5)
    ref.check(out[:qb[-1]], o[:qb[-1]], slack[:qb[-1]], "skewed")
    ws = gpu_lib.attention_workspace(q.shape[0], k.shape[0], len(lq), hq, hkv, d)
    ws.fill_(255)
    again = torch.full_like(q, -7.0)
    gpu_lib.attention(q, k, v, ints(qb), ints(kb), causal=causal, out=again, workspace=ws)
    assert torch.equal(again, out)


def test_attention_bad_offsets_by_length(gpu_lib):
    """Offsets that name the same rows again and again, in calls that split by length: nothing outside the tensor
    or behind the workspace is written."""
    import torch
    randn = gen(43)
    q, k, v = randn(20, 4, 64).half(), randn(9000, 2, 64).half(), randn(9000, 2, 64).half()
    need = gpu_lib.attention_workspace(20, 9000, 6, 4, 2, 64).numel()
    for qo, ko in (([0, 20, 0, 20, 0, 20, 0], [0, 9000, 0, 9000, 0, 9000, 0]), ([0, 20, 0, 20, 0, 20, 0], [0, 9000, 10, 20, 5, 9000, 1]),
                   ([-5, 30, 2, 2**31 - 1, -2**31, 20, 20], [9000, 0, 9000, 0, 2**31 - 1, -2**31, 9000])):
        for causal in (False, True):
            guard = torch.full((60, 4, 64), -7.0, device="cuda", dtype=torch.float16)
            ws = torch.full((4 * need,), 255, dtype=torch.uint8, device="cuda")
            gpu_lib.attention(q, k, v, ints(qo), ints(ko), out=guard[20:40], causal=causal, workspace=ws[:need])
            assert (guard[:20] == -7).all() and (guard[40:] == -7).all() and (ws[need:] == 255).all()


def test_attention_many_samples(gpu_lib):
    """More samples than a wave has lanes, unequal and some empty, few and many rows each; the longest samples
    first or last."""
    import torch
    for lens in ([(1 + i % 5, 3 + 7 * i % 50) for i in range(150)], [(100, 300 - 18 * i) for i in range(16)], [(64, 20 * i) for i in range(17)],
                 [(i % 3 * 90, 200 + 40 * i) for i in range(9)]):
        randn = gen(len(lens))
        qb, kb = ref.offsets_of([a for a, _ in lens]), ref.offsets_of([b for _, b in lens])
        q, k, v = randn(qb[-1], 4, 64).half(), randn(kb[-1], 2, 64).half(), randn(kb[-1], 2, 64).half()
        for causal in (False, True):
            out = gpu_lib.attention(q, k, v, ints(qb), ints(kb), causal=causal)
            o, slack = ref.attention(q, k, v, qb, kb, causal, 0.125)
            ref.check(out, o, slack, f"{len(lens)} samples")


def test_attention_minus_infinity(gpu_lib):
    """Scores of -inf beside finite ones weigh nothing; a row of nothing but -inf is 0/0 = NaN as in the
    formula, and a row that sees no key is zero."""
    import torch
    q = torch.ones(4, 1, 8, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(200, 1, 8, device="cuda", dtype=torch.bfloat16)
    v = torch.arange(200, device="cuda").bfloat16()[:, None, None].expand(200, 1, 8).contiguous()
    k[:100, 0, 0] = -math.inf
    k[199, 0, 0] = -math.inf
    out = gpu_lib.attention(q, k, v)
    o, slack = ref.attention(q, k, v, [0, 4], [0, 200], False, 8 ** -0.5)
    ref.check(out, o, slack, "-inf")
    assert torch.isnan(gpu_lib.attention(q, k[:100], v[:100])).all()
    out = gpu_lib.attention(q, k[100:102], v[100:102], causal=True)
    assert (out[:2] == 0).all() and (out[2, 0] == 100).all() and torch.isfinite(out).all()


def test_attention_leaves_other_rows(gpu_lib):
    """Rows of out outside the samples keep what they held, also where offsets are out of order or range."""
    import torch
    randn = gen(14)
    q, k, v = (randn(200, 2, 64).half() for _ in range(3))
    out = torch.full((200, 2, 64), -7.0, device="cuda", dtype=torch.float16)
    gpu_lib.attention(q, k, v, ints([5, 50, 180]), ints([0, 100, 200]), out=out)
    assert (out[:5] == -7).all() and (out[180:] == -7).all()
    o, slack = ref.attention(q, k, v, [5, 50, 180], [0, 100, 200], False, 0.125)
    ref.check(out[5:180], o[5:180], slack[5:180], "rows")
    for qo, ko in (([-9, 60, 900], [0, 5000, 7]), ([150, 10, 200], [200, -4, 2**31 - 1]), ([2**31 - 1, -2**31, 3], [0, 1, 2])):
        guard = torch.full((400, 2, 64), -7.0, device="cuda", dtype=torch.float16)
        gpu_lib.attention(q, k, v, ints(qo), ints(ko), out=guard[100:300], causal=True)
        assert (guard[:100] == -7).all() and (guard[300:] == -7).all()


@pytest.mark.parametrize("lo,hi,lk", [(2, 4, 9000), (1, 2, 30), (3, 300, 700), (5, 5, 100)])
def test_attention_one_sample_inside(gpu_lib, lo, hi, lk):
    """One sample that begins behind the first row and ends before the last, its keys split or not."""
    import torch
    randn = gen(lo)
    q, k, v = randn(hi + 4, 4, 128).bfloat16(), randn(lk + 20, 2, 128).bfloat16(), randn(lk + 20, 2, 128).bfloat16()
    k[:7], v[:7], k[7 + lk:], v[7 + lk:] = math.nan, math.inf, math.nan, math.nan
    for causal in (False, True):
        out = torch.full_like(q, -7.0)
        gpu_lib.attention(q, k, v, ints([lo, hi]), ints([7, 7 + lk]), causal=causal, out=out)
        assert (out[:lo] == -7).all() and (out[hi:] == -7).all()
        o, slack = ref.attention(q[lo:hi], k[7:7 + lk], v[7:7 + lk], [0, hi - lo], [0, lk], causal, 128 ** -0.5)
        ref.check(out[lo:hi], o, slack, "inside")


def test_attention_many_rows(gpu_lib):
    """More units than the device's rounds by far, and a last one of a single row."""
    randn = gen(16)
    q, k, v = randn(200_001, 2, 64).half(), randn(70, 1, 64).half(), randn(70, 1, 64).half()
    o, slack = ref.attention(q, k, v, [0, 200_001], [0, 70], False, 0.125)
    ref.check(gpu_lib.attention(q, k, v), o, slack, "many rows")


def test_many_tiny_samples(gpu_lib):
    """Two thousand samples of 0 to 2 rows."""
    import torch
    lens = [i % 3 for i in range(2000)]
    bounds = ref.offsets_of(lens)
    randn = gen(17)
    x = randn(bounds[-1], 64)
    y, slack = ref.group_norm(x, 8, bounds, None, None, 1e-5, False)
    ref.check(gpu_lib.group_norm(x, 8, eps=1e-5, offsets=ints(bounds)), y, slack, "norm")
    q = x.view(-1, 1, 64).half()
    out = gpu_lib.attention(q, q, q, ints(bounds), ints(bounds), causal=True)
    first = torch.tensor([a for a, m in zip(bounds, lens) if m], device="cuda")
    assert torch.equal(out[first], q[first])       # a sample's first row sees itself alone
    o, slack = ref.attention(q, q, q, bounds[:302], bounds[:302], True, 0.125)
    ref.check(out[:bounds[301]], o[:bounds[301]], slack[:bounds[301]], "attention")


def test_attention_cache_past_32_bits(gpu_lib):
    """A cache whose rows lie more than 4 GiB apart: one new token, and a prompt, at its end."""
    import torch
    randn = gen(15)
    rows, stride = 2200, 1 << 20
    big = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    kv = big.view(rows, stride)[:, : 2 * 64].view(rows, 2, 64)
    data = randn(rows, 2, 64).bfloat16()
    kv.copy_(data)
    for nq in (1, 100):
        q = randn(nq, 1, 64).bfloat16()
        out = gpu_lib.attention(q, kv[:, :1], kv[:, 1:], causal=True)
        o, slack = ref.attention(q, data[:, :1], data[:, 1:], [0, nq], [0, rows], True, 0.125)
        ref.check(out, o, slack, f"{nq} rows")


def test_attention_f32_views(gpu_lib):
    """fp32 heads as views into one linear's output, and more rows than one workgroup's."""
    import torch
    randn = gen(41)
    qkv = randn(333, 3, 4, 72)
    q, k, v = qkv.unbind(1)
    out = torch.full((333, 4, 80), -7.0, device="cuda")
    gpu_lib.attention(q, k, v, causal=True, out=out[:, :, 8:])
    o, slack = ref.attention(q, k, v, [0, 333], [0, 333], True, 72 ** -0.5)
    ref.check(out[:, :, 8:], o, slack, "f32 views")
    assert (out[:, :, :8] == -7).all()


def test_attention_empty(gpu_lib):
    import torch
    q = torch.zeros(0, 2, 64, device="cuda", dtype=torch.float16)
    k = torch.ones(9, 2, 64, device="cuda", dtype=torch.float16)
    assert gpu_lib.attention(q, k, k).shape == (0, 2, 64)
    assert (gpu_lib.attention(k, q, q) == 0).all()
    assert (gpu_lib.attention(k, q, q, ints([0, 4, 9]), ints([0, 0, 0]), causal=True) == 0).all()


# ---- streams, graphs, a block -------------------------------------------------------------------
def _calls(pkg, torch, n, seed):
    """The three operators on fixed buffers: what a captured step holds."""
    randn = gen(seed)
    x, gamma = randn(n, 64), 1 + 0.1 * randn(64)
    q, k, v = (randn(n, 4, 64).bfloat16() for _ in range(3))
    one = randn(2, 4, 64).bfloat16()
    pos = torch.randint(0, 64, (n, 3), device="cuda", dtype=torch.int32)
    offs, qoffs = ints([0, n // 3, n]), ints([0, 1, 2])
    outs = [torch.empty_like(x), torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty_like(one)]
    ws = [pkg.group_norm_workspace(n, 64, 8, 2), pkg.attention_workspace(n, n, 2, 4, 4, 64), pkg.attention_workspace(2, n, 2, 4, 4, 64)]

    def call(stream=None):
        pkg.group_norm(x, 8, gamma, silu=True, offsets=offs, out=outs[0], workspace=ws[0], stream=stream)
        pkg.rope_axes(q, pos, k=k, q_out=outs[1], k_out=outs[2], stream=stream)
        pkg.attention(outs[1], outs[2], v, offs, offs, out=outs[3], workspace=ws[1], stream=stream)
        pkg.attention(one, outs[2], v, qoffs, offs, causal=True, out=outs[4], workspace=ws[2], stream=stream)
    return call, (x, q, k, v, one), outs


@pytest.mark.parametrize("n", [300, 9000])
def test_captured_and_replayed(gpu_lib, n):
    """A captured step replayed with new inputs in between gives the eager result each time."""
    import torch
    call, inputs, outs = _calls(gpu_lib, torch, n, 21)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(4):
        for t in inputs:
            t.copy_(torch.randn_like(t))
        for o in outs:
            o.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for o in outs:
            o.fill_(math.nan)
        call()
        torch.cuda.synchronize()
        for a, b in zip(got, outs):
            assert torch.equal(a, b), f"replay {step}"


def test_other_stream(gpu_lib):
    """The same on a stream of its own, given as an argument or made current, and two of them at once."""
    import torch
    call, _, outs = _calls(gpu_lib, torch, 5000, 22)
    call2, _, outs2 = _calls(gpu_lib, torch, 5000, 23)
    call()
    call2()
    torch.cuda.synchronize()
    want, want2 = [o.clone() for o in outs], [o.clone() for o in outs2]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for o in outs + outs2:
        o.fill_(math.nan)
    torch.cuda.synchronize()
    call(s1)
    with torch.cuda.stream(s2):
        call2()
    torch.cuda.synchronize()
    for a, b in zip(outs + outs2, want + want2):
        assert torch.equal(a, b)
    # buffers made by the call on the given stream
    q = torch.randn(700, 2, 64, device="cuda").half()
    torch.cuda.synchronize()
    a = gpu_lib.attention(q, q, q, stream=s1)
    b = gpu_lib.group_norm(q.view(700, 128), 4, stream=s1)
    c = gpu_lib.rope_axes(q, torch.zeros(700, 1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(a, gpu_lib.attention(q, q, q)) and torch.equal(b, gpu_lib.group_norm(q.view(700, 128), 4)) and torch.equal(c, q)


@pytest.mark.parametrize("key", ["f16", "bf16"])
def test_block(gpu_lib, key):
    """Group norm with SiLU, the linear to q, k and v, rotary positions, attention, the output linear with
    the residual: each step against its 64-bit form on the input it got."""
    import torch
    pkg, randn = gpu_lib, gen(31)
    n, c, heads, d, dt = 1300, 256, 4, 64, dtype(key)
    bounds = [0, 500, 501, 1300]
    offs = ints(bounds)
    x, gamma, beta = randn(n, c), 1 + 0.1 * randn(c), 0.1 * randn(c)
    wqkv, bqkv = (randn(3 * c, c) / 16).to(dt), 0.1 * randn(3 * c)
    wo, bo = (randn(c, c) / 16).to(dt), 0.1 * randn(c)
    gq, gk = 1 + 0.1 * randn(heads, d), 1 + 0.1 * randn(heads, d)
    pos = torch.randint(0, 64, (n, 3), device="cuda", dtype=torch.int32)
    h = pkg.group_norm(x, 32, gamma, beta, silu=True, offsets=offs, out_dtype=dt)
    y, slack = ref.group_norm(x, 32, bounds, gamma, beta, 1e-6, True)
    ref.check(h, y, slack, "norm")
    qkv = pkg.linear(h, wqkv, bqkv).view(n, 3, heads, d)
    q, k, v = qkv.unbind(1)
    q0, k0 = q.clone(), k.clone()
    pkg.rope_axes(q, pos, k=k, q_gamma=gq, k_gamma=gk, q_out=q, k_out=k)
    for a, b, g in ((q, q0, gq), (k, k0, gk)):
        y, slack = ref.rope(b, pos, [10, 10, 10], 10000.0, True, g, 1e-6)
        ref.check(a, y, slack, "rope")
    o = pkg.attention(q, k, v, offs, offs)
    y, slack = ref.attention(q, k, v, bounds, bounds, False, d ** -0.5)
    ref.check(o, y, slack, "attention")
    out = pkg.linear_ex(o.view(n, c), wo, bo, residual=x, out_dtype=torch.float32)
    want = o.view(n, c).double() @ wo.double().t() + bo.double() + x.double()
    assert ((out.double() - want).abs().max() / want.abs().max()).item() < 1e-5
