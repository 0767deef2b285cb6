"""GPU tests of a served block's pieces: rms_norm, mx_quantize, linear_mx, the paged cache and attention_cached against
their 64-bit forms, at the sizes, masks, strides, pages and values where they can go wrong; streams, captured graphs, and
a run of them together."""
from __future__ import annotations

import math

import pytest

import served_ref as sr
import transformer_ref as ref

pytestmark = pytest.mark.gpu


def dtype(key):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "mx8": torch.float8_e4m3fn}[key]


def gen(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *shape: torch.randn(shape, generator=g, device="cuda")


def ints(values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def same(a, b):
    """Equal bits."""
    import torch
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- numbers of few bits ------------------------------------------------------------------------
@pytest.mark.parametrize("n,c", [(1, 32), (3, 64), (7, 96), (130, 1024), (5, 4128)])
@pytest.mark.parametrize("key", ["f32", "f16", "bf16"])
def test_mx_quantize(gpu_lib, n, c, key):
    """Bit for bit: blocks of every size of values, of powers of two and halfway cases, of zeros, and with an Inf or a NaN."""
    import torch
    print(f"[mx_quantize] {n} x {c} {key}", flush=True)
    randn = gen(n * c)
    x = randn(n, c) * torch.exp2(torch.floor(randn(n, c // 32).repeat_interleave(32, 1) * (40 if key != "f16" else 3)))
    flat = x.view(-1, 32)
    flat[0] = torch.arange(32, device="cuda") * 0.0625 + 0.03125       # halfway between codes
    if len(flat) > 1:
        flat[1, :] = 0
    if len(flat) > 2:
        flat[2, 3] = math.inf
        flat[-1, 31] = math.nan
    x = x.to(dtype(key))
    out = gpu_lib.mx_quantize(x)
    codes, powers = sr.to_mx(x)
    assert out.codes.dtype == torch.float8_e4m3fn and out.powers.dtype == torch.float8_e8m0fnu
    assert same(out.powers, powers)
    fine = (powers.view(torch.uint8) != 255).repeat_interleave(32, 1)
    assert torch.equal(out.codes.float()[fine], codes.float()[fine])
    # nothing is off by more than half a step of its value, or of the smallest step
    y, v = sr.of_mx(out), x.double()
    s = sr.scale_of(powers.view(torch.uint8)).repeat_interleave(32, 1)
    assert bool(((y - v).abs() <= torch.maximum(v.abs() * 2.0 ** -4, s * 2.0 ** -10))[fine].all())
    assert bool(torch.isnan(y[~fine]).all())


# ---- RMS norm -----------------------------------------------------------------------------------
RMS_CASES = [(1, 1), (1, 8), (3, 7), (5, 32), (1, 1024), (9, 100), (33, 512), (70, 520), (17, 2048), (6, 2056), (5, 4096),
             (3, 8192), (2, 8224), (2, 20_000), (9001, 96), (8300, 1000), (9, 500), (8193, 516),
             (5, 1028), (4099, 1500), (3, 4092), (8195, 501), (7, 999), (4097, 1027), (2, 4095), (3, 4100), (2, 5001)]


@pytest.mark.parametrize("n,c", RMS_CASES)
@pytest.mark.parametrize("xk,rk,ok", [("f32", None, "f32"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f16"), ("bf16", "f32", "f32"),
                                      ("f32", "f16", "bf16")])
def test_rms_norm(gpu_lib, n, c, xk, rk, ok):
    import torch
    print(f"[rms norm] {n} x {c} {xk}+{rk}->{ok}", flush=True)
    randn = gen(n + c)
    x = (randn(n, c) * (0.1 + randn(n, 1).abs())).to(dtype(xk))
    r = None if rk is None else (randn(n, c) * 3).to(dtype(rk))
    gamma = None if n % 2 == 0 else 1 + 0.3 * randn(c)
    out = gpu_lib.rms_norm(x, gamma, eps=1e-5, residual=r, out_dtype=dtype(ok))
    y, h = sr.rms_norm(x, r, gamma, 1e-5)
    if rk is not None:
        out, ro = out
        assert ro.dtype == dtype(rk)
        ref.check(ro, h, h.abs() * 2.0 ** -24, "residual")
    assert out.dtype == dtype(ok)
    ref.check(out, y, y.abs() * sr.NORM_SLACK, "rms norm")


def check_mx(out, y, what):
    """An Mx against values in 64 bits that the kernel knows to NORM_SLACK of themselves: every power and code is that of a
    value that near."""
    import torch
    codes, powers = out
    amax, power = sr.amax_of(y), powers.view(torch.uint8)
    lo, hi = sr.power_of(amax * (1 - sr.NORM_SLACK), 448.0), sr.power_of(amax * (1 + sr.NORM_SLACK), 448.0)
    assert bool(((power == lo) | (power == hi)).all()), f"{what}: powers"
    fine = (power != 255).repeat_interleave(32, -1)
    s = sr.scale_of(power).repeat_interleave(32, -1)
    z = y.double() / s
    a, b = sr.round_e4m3((z.abs() * (1 - sr.NORM_SLACK)).clamp(max=448)), sr.round_e4m3((z.abs() * (1 + sr.NORM_SLACK)).clamp(max=448))
    v = codes.double()
    ok = ((v.abs() == a) | (v.abs() == b)) & ((v == 0) | (torch.sign(v) == torch.sign(y)))
    assert bool(ok[fine].all()), f"{what}: {int((~ok[fine]).sum())} codes"


@pytest.mark.parametrize("n,c", [(1, 32), (5, 1024), (33, 512), (70, 544), (17, 2048), (5, 4128), (3, 8192), (2, 8224), (8300, 96)])
@pytest.mark.parametrize("xk,rk", [("f32", None), ("bf16", "bf16"), ("f16", "f32")])
def test_rms_norm_mx(gpu_lib, n, c, xk, rk):
    print(f"[rms norm, 8 bits] {n} x {c} {xk}+{rk}", flush=True)
    randn = gen(n + c)
    x = (randn(n, c) * (0.1 + randn(n, 1).abs())).to(dtype(xk))
    r = None if rk is None else (randn(n, c) * 3).to(dtype(rk))
    gamma = 1 + 0.3 * randn(c)
    out = gpu_lib.rms_norm(x, gamma, residual=r, out_dtype=dtype("mx8"))
    y, h = sr.rms_norm(x, r, gamma, 1e-6)
    if rk is not None:
        out, ro = out
        ref.check(ro, h, h.abs() * 2.0 ** -24, "residual")
    check_mx(out, y, "8 bits")


@pytest.mark.parametrize("n,c", [(3, 96), (9, 544), (8300, 1024), (5, 2080), (2, 4096), (2, 4128)])
def test_rms_norm_mx_off_a_boundary(gpu_lib, n, c):
    """Rows off a 16-byte boundary, value by value, into 8 bits."""
    import torch
    randn = gen(n + c)
    x = torch.empty(n * c + 1, dtype=torch.bfloat16, device="cuda")[1:].view(n, c).copy_(randn(n, c) * 2)
    gamma = 1 + 0.3 * randn(c)
    out = gpu_lib.rms_norm(x, gamma, out_dtype=dtype("mx8"))
    check_mx(out, sr.rms_norm(x, None, gamma, 1e-6)[0], "8 bits")


def test_rms_norm_places(gpu_lib):
    """Outputs in the inputs' place, rows off a 16-byte boundary, strided rows and values that are not finite."""
    import torch
    randn = gen(5)
    x, r, gamma = randn(40, 256).bfloat16(), randn(40, 256), 1 + 0.2 * randn(256)
    y0, r0 = gpu_lib.rms_norm(x, gamma, residual=r)
    xi, ri = x.clone(), r.clone()
    y1, r1 = gpu_lib.rms_norm(xi, gamma, residual=ri, out=xi, residual_out=ri)
    assert y1 is xi and r1 is ri and torch.equal(xi, y0) and torch.equal(ri, r0)
    for c in (256, 20_000):     # (read once, and twice)
        a, b = randn(3, c).half(), randn(3, c).half()
        want = gpu_lib.rms_norm(a, residual=b)
        b1 = b.clone()
        got = gpu_lib.rms_norm(a, residual=b1, out=b1, residual_out=torch.empty_like(b))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty(40 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(40, 256).copy_(x)
    y2, r2 = gpu_lib.rms_norm(odd, gamma, residual=r)
    ref.check(y2, *[(t, t.abs() * sr.NORM_SLACK) for t in [sr.rms_norm(x, r, gamma, 1e-6)[0]]][0], "unaligned")
    assert torch.equal(gpu_lib.rms_norm(x.t().contiguous().t(), gamma, residual=r)[0], y0)
    bad = randn(4, 64)
    bad[1, 5], bad[2, 7] = math.nan, math.inf
    y = gpu_lib.rms_norm(bad)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[[0, 3]]).all())
    assert bool((y[2] == 0).sum() == 63) and math.isnan(y[2, 7])        # Inf / Inf, and the others over Inf
    m = gpu_lib.rms_norm(bad, out_dtype=torch.float8_e4m3fn)
    assert m.powers.view(torch.uint8)[1].tolist() == [255, 255] and m.powers.view(torch.uint8)[2, 0] == 255
    z = gpu_lib.rms_norm(torch.zeros(2, 64, device="cuda"), out_dtype=torch.float8_e4m3fn)
    assert bool((sr.of_mx(z) == 0).all())
    assert gpu_lib.rms_norm(randn(0, 64)).shape == (0, 64)


# ---- linear -------------------------------------------------------------------------------------
LINEAR_CASES = [(1, 32, 1), (1, 1024, 64), (5, 96, 27), (3, 160, 100), (16, 128, 16), (17, 512, 333), (64, 2048, 72), (65, 256, 1000), (128, 1056, 130),
                (200, 32, 7), (257, 640, 260), (1000, 1024, 1000), (515, 4096, 520), (2606, 768, 256), (3001, 2048, 2500), (3001, 2080, 2500), (20000, 480, 1000), (9, 96, 8200), (29, 544, 5000), (45, 1024, 300), (9, 1024, 5000),
                (1500, 1024, 1500), (1500, 1056, 1500), (12001, 1024, 1001), (12001, 1056, 1001), (13001, 1024, 1000), (13001, 1056, 1000),
                (12001, 1024, 1004), (13001, 4096, 1000)]


@pytest.mark.parametrize("n,ci,co", LINEAR_CASES)
@pytest.mark.parametrize("ok,act,extra", [("f32", "none", True), ("bf16", "silu", False), ("f16", "none", True), ("f32", "silu", False)])
def test_linear_mx(gpu_lib, n, ci, co, ok, act, extra):
    print(f"[linear] {n} x {ci} -> {co} {ok} {act}", flush=True)
    randn = gen(n + ci + co)
    x = gpu_lib.Mx(*sr.to_mx(randn(n, ci) * (1 + randn(n, 1).abs())))
    w = gpu_lib.Mx(*sr.to_mx(randn(co, ci) / math.sqrt(ci)))
    bias, res = (0.3 * randn(co), randn(n, co)) if extra else (None, None)
    out = gpu_lib.linear_mx(x, w, bias, act=act, residual=res, out_dtype=dtype(ok))
    assert out.dtype == dtype(ok)
    y, slack = sr.linear(sr.of_mx(x), sr.of_mx(w), bias, act, res, ok == "f32")
    ref.check(out, y, slack, "linear")


@pytest.mark.parametrize("n", [3, 40, 300])
@pytest.mark.parametrize("ok", ["f32", "bf16"])
def test_linear_mx_values(gpu_lib, n, ok):
    """NaN powers reach their rows and outputs alone; powers far apart; the residual's own place."""
    import torch
    randn = gen(n)
    xc, xp = sr.to_mx(randn(n, 256))
    wc, wp = sr.to_mx(randn(96, 256) / 16)
    y0 = gpu_lib.linear_mx((xc, xp), (wc, wp), out_dtype=dtype(ok))
    xp1, wp1 = xp.clone(), wp.clone()
    xp1.view(torch.uint8)[2, 5] = 255
    wp1.view(torch.uint8)[17, 0] = 255
    y = gpu_lib.linear_mx((xc, xp1), (wc, wp1), out_dtype=dtype(ok))
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[:, 17]).all())
    keep_r, keep_c = [i for i in range(n) if i != 2], [i for i in range(96) if i != 17]
    assert torch.equal(y[keep_r][:, keep_c], y0[keep_r][:, keep_c])
    xp2, wp2 = xp.clone(), wp.clone()      # 2^100 times x, 2^-100 times W
    xp2.view(torch.uint8).add_(100)
    wp2.view(torch.uint8).sub_(100)
    assert torch.equal(gpu_lib.linear_mx((xc, xp2), (wc, wp2), out_dtype=dtype(ok)), y0)
    if ok == "f32":
        res = randn(n, 96)
        want = gpu_lib.linear_mx((xc, xp), (wc, wp), residual=res, out_dtype=dtype(ok))
        got = gpu_lib.linear_mx((xc, xp), (wc, wp), residual=res, out=res)
        assert got is res and torch.equal(got, want)
    out = torch.full((n, 97), 7.0, device="cuda", dtype=dtype(ok)).view(-1)[1: 1 + n * 96].view(n, 96)      # off a boundary
    assert torch.equal(gpu_lib.linear_mx((xc, xp), (wc, wp), out=out), y0)


def test_linear_mx_empty(gpu_lib):
    x, w = gpu_lib.mx_empty(0, 64), gpu_lib.mx_empty(8, 64)
    assert gpu_lib.linear_mx(x, w).shape == (0, 8)


# ---- the cache ----------------------------------------------------------------------------------
def make_cache(pkg, lengths, page, heads, d, held, seed, spare=2, fill=True):
    """A cache whose samples' pages are dealt at random, and its table; its contents are rounded random values."""
    import torch
    counts = [-(-m // page) for m in lengths]
    pool = sum(counts) + spare
    cache = pkg.kv_cache(pool, page, heads, d, "mx4" if held == "mx4" else dtype(held))
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(counts))), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(counts):
        table[i, :m] = order[at: at + m]
        at += m
    table = table.cuda()
    if fill and sum(lengths):
        randn = gen(seed + 1)
        n = sum(lengths)
        k, v = randn(n, heads, d) * (0.2 + randn(n, 1, 1).abs()), randn(n, heads, d)
        pkg.kv_append(cache, k.to(dtype("bf16")), v.to(dtype("bf16")), table, ints(lengths), offsets=ints(ref.offsets_of(lengths)))
    return cache, table


APPEND_CASES = [
    # new rows, lengths after them, hq, hkv, d, page, axes, pairs
    ([1], [1], 4, 2, 64, 16, 1, None), ([1], [70], 8, 1, 128, 64, 1, None), ([5], [5], 1, 1, 8, 16, 2, None),
    ([3, 0, 1, 40], [3, 9, 17, 100], 6, 3, 80, 32, 3, [10, 12, 8]), ([1] * 20, list(range(1, 21)), 8, 4, 96, 16, 1, None),
    ([130, 7], [130, 300], 8, 8, 32, 256, 3, None), ([64], [64], 16, 2, 128, 128, 2, [16, 40]), ([9, 9], [40, 9], 2, 2, 24, 16, 1, [5]),
    ([33], [50], 3, 1, 72, 16, 1, None), ([300], [1000], 5, 5, 120, 32, 0, None), ([11, 2], [11, 2], 4, 4, 40, 16, 4, [1, 2, 3, 4]),
]


@pytest.mark.parametrize("case", range(len(APPEND_CASES)))
@pytest.mark.parametrize("held,key", [("mx4", "bf16"), ("mx4", "f16"), ("mx4", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("norm,interleaved", [(True, True), (False, False), (True, False)])
def test_append_and_gather(gpu_lib, case, held, key, norm, interleaved):
    import torch
    new, lengths, hq, hkv, d, page, axes, pairs = APPEND_CASES[case]
    print(f"[append] {case} held {held} {key} norm={norm} interleaved={interleaved}", flush=True)
    randn, n = gen(case), sum(new)
    q, k, v = randn(n, hq, d).to(dtype(key)), randn(n, hkv, d).to(dtype(key)), randn(n, hkv, d).to(dtype(key))
    gq, gk = (1 + 0.2 * randn(hq, d), 1 + 0.2 * randn(hkv, d)) if norm else (None, None)
    pos = torch.randint(0, 100_000, (n, axes), device="cuda", dtype=torch.int32) if axes else None
    pairs = pairs or ([d // 2 // axes] * axes if axes else [])
    cache, table = make_cache(gpu_lib, lengths, page, hkv, d, held, case)
    before = [t.clone() for t in sr.decode(cache)]
    b = ref.offsets_of(new)
    qo = gpu_lib.kv_append(cache, k, v, table, ints(lengths), offsets=ints(b), q=q, pos=pos, pairs=pairs if axes else None,
                           theta=5000.0, interleaved=interleaved, q_gamma=gq, k_gamma=gk, eps=1e-5)
    zero = torch.zeros((n, 1), dtype=torch.int32, device="cuda")
    yq, sq = ref.rope(q, pos if axes else zero, pairs, 5000.0, interleaved, gq, 1e-5)
    yk, sk = ref.rope(k, pos if axes else zero, pairs, 5000.0, interleaved, gk, 1e-5)
    ref.check(qo, yq, sq, "q")
    after = sr.decode(cache)
    rows = []
    for s, (a, m) in enumerate(zip(b, new)):
        rows += [(a + i, *sr.place(cache, table, s, lengths[s] - m + i)) for i in range(m)]
    r, p, t = (torch.tensor(x, device="cuda") for x in zip(*rows))
    if held == "mx4":
        # (the reference turns in 64 bits as well: a code differs only within some 2^-50 of a border)
        assert torch.equal(after[0][p, t], sr.mx4_values(yk)[r]) and torch.equal(after[1][p, t], sr.mx4_values(v)[r])
    else:
        # (ref.check wants the type that was rounded to)
        ref.check(after[0][p, t].to(dtype(held)), yk[r], sk[r], "k")
        assert torch.equal(after[1][p, t], v.to(dtype(held)).double()[r])
    # the other slots hold what they held
    for x, y in zip(before, after):
        x[p, t] = 0
        y[p, t] = 0
        assert torch.equal(x, y)
    after = sr.decode(cache)
    ko, vo = gpu_lib.kv_gather(cache, table, ints(lengths), offsets=ints(b), n=n, out_dtype=torch.float32)
    assert torch.equal(ko.double()[r], after[0][p, t]) and torch.equal(vo.double()[r], after[1][p, t])
    if held == "mx4":
        ko, vo = gpu_lib.kv_gather(cache, table, ints(lengths), offsets=ints(b), n=n)
        assert ko.dtype == torch.bfloat16 and torch.equal(ko.double()[r], after[0][p, t]) and torch.equal(vo.double()[r], after[1][p, t])


def test_append_places(gpu_lib):
    """Rows of no sample, keys that the table does not reach, pages that are not the pool's, strided views, q in place."""
    import torch
    for held in ("mx4", "bf16"):
        randn = gen(3)
        cache, table = make_cache(gpu_lib, [40, 30], 16, 2, 64, held, 9)
        table[0, 1] = cache.pages           # keys 16..31 of sample 0: nowhere
        table[1, 0] = -5                    # keys 0..15 of sample 1
        before = cache.data.clone()
        qkv = randn(60, 8, 64).bfloat16()   # q, k and v in one tensor
        q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
        offs, lengths = [5, 45, 55], [50, 7]        # 40 rows to keys 10..49 (48 and 49 past the table), 10 to -3..6
        want = gpu_lib.kv_append(cache, k, v, table, ints(lengths), offsets=ints(offs), q=q)
        written = cache.data.clone()
        keys = {**{(0, 10 + i): 5 + i for i in range(40)}, **{(1, i - 3): 45 + i for i in range(10)}}
        kd, vd = sr.decode(cache)
        kb, vb = sr.decode(gpu_lib.KVCache(before, 16, 2, 64, cache.dtype))
        val = sr.mx4_values if held == "mx4" else lambda x: x.double()
        n_held = 0
        for (s, j), row in keys.items():
            at = sr.place(cache, table, s, j)
            if at:
                n_held += 1
                kb[at], vb[at] = val(k)[row], val(v)[row]
        assert n_held == 22 and torch.equal(kd, kb) and torch.equal(vd, vb)
        # in place, and rows of no sample left
        cache.data.copy_(before)
        mark = qkv.clone()
        got = gpu_lib.kv_append(cache, k, v, table, ints(lengths), offsets=ints(offs), q=q, q_out=q)
        assert got.data_ptr() == q.data_ptr() and torch.equal(got[5:55], want[5:55]) and same(cache.data, written)
        assert torch.equal(qkv[:5], mark[:5]) and torch.equal(qkv[55:], mark[55:]) and torch.equal(qkv[:, 4:], mark[:, 4:])
        # out again: zeros where nothing is held
        ko = torch.full((60, 2, 64), 7.0, device="cuda")
        vo = torch.full((60, 3, 64), 7.0, device="cuda")[:, 1:]
        gpu_lib.kv_gather(cache, table, ints(lengths), offsets=ints(offs), k_out=ko, v_out=vo)
        assert bool((ko[:5] == 7).all() and (ko[55:] == 7).all() and (vo[55:] == 7).all())
        for (s, j), row in keys.items():
            at = sr.place(cache, table, s, j)
            assert torch.equal(ko[row].double(), kb[at] if at else torch.zeros_like(kb[0, 0]))
            assert torch.equal(vo[row].double(), vb[at] if at else torch.zeros_like(vb[0, 0]))
        # offsets out of order or of the tensor stay inside it
        gpu_lib.kv_append(cache, k, v, table, ints([50, 7]), offsets=ints([30, -4, 1 << 30]), q=q)
        gpu_lib.kv_gather(cache, table, ints([-3, 1 << 30]), offsets=ints([30, -4, 1 << 30]), n=60)
        torch.cuda.synchronize()


def test_append_far_positions(gpu_lib):
    """Positions up to 2^28: the codes are still those of 64-bit angles, to the angles' own 2^-24."""
    import torch
    n = 400
    cache = gpu_lib.kv_cache(25, 16, 1, 128)
    table = torch.arange(25, dtype=torch.int32, device="cuda").view(1, 25)
    k = gen(1)(n, 1, 128)
    pos = (torch.arange(n, device="cuda", dtype=torch.int32) * 671_088)[:, None].contiguous()
    gpu_lib.kv_append(cache, k, k, table, ints([n]), pos=pos)
    y, _ = ref.rope(k, pos, [64], 10000.0, True, None, 1e-6)
    kd = sr.keys_of(cache, table, [n], 0)[0]
    # between the codes of values that much smaller and larger
    lo, hi = (sr.mx4_values(y * (1 + e)) for e in (-(2.0 ** -20), 2.0 ** -20))
    assert bool(((kd == lo) | (kd == hi) | ((kd - y).abs() <= (sr.mx4_values(y) - y).abs() + 2.0 ** -18 * y.abs().amax())).all())


def test_append_values(gpu_lib):
    """Blocks with Inf or NaN, of zeros, and of halfway values."""
    import torch
    cache = gpu_lib.kv_cache(2, 16, 1, 64)
    k, v = torch.zeros(3, 1, 64, device="cuda"), torch.zeros(3, 1, 64, device="cuda")
    k[0, 0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6] * 4, device="cuda") * 2.0 ** -40
    k[1, 0, 40] = math.inf
    v[1, 0, 3] = math.nan
    v[2, 0, 0] = 3.4e38
    table = ints([[1]])
    gpu_lib.kv_append(cache, k, v, table, ints([3]))
    kd, vd = sr.decode(cache)
    assert torch.equal(kd[1, 0, 0], sr.mx4_values(k[0])[0]) and bool((kd[1, 0, 0, 32:] == 0).all())
    assert bool(torch.isnan(kd[1, 1, 0, 32:]).all()) and bool((kd[1, 1, 0, :32] == 0).all())
    assert bool(torch.isnan(vd[1, 1, 0, :32]).all()) and vd[1, 2, 0, 0].item() == sr.mx4_values(v[2])[0, 0].item()
    ko, _ = gpu_lib.kv_gather(cache, table, ints([3]), n=3, out_dtype=torch.float32)
    assert bool(torch.isnan(ko[1, 0, 32:]).all())


# ---- attention to it ----------------------------------------------------------------------------
ATTEND_CASES = [
    # new rows, keys, hq, hkv, d, page
    ([1], [1], 1, 1, 8, 16), ([1], [31], 4, 4, 64, 16), ([1], [33], 8, 1, 128, 16), ([1], [4000], 16, 2, 128, 64), ([1, 1, 1], [5, 0, 700], 8, 2, 96, 32),
    ([3, 0, 2], [3, 10, 64], 6, 2, 80, 16), ([8] * 5, [8, 100, 33, 257, 9], 8, 8, 32, 128), ([5], [3], 4, 2, 64, 16), ([17], [200], 2, 1, 128, 256),
    ([100], [100], 4, 4, 64, 32), ([40, 70, 1], [300, 70, 2], 12, 4, 128, 64), ([300], [1000], 8, 1, 40, 16), ([1] * 70, [(i * 37) % 211 for i in range(70)], 4, 1, 64, 32),
    ([129], [129], 3, 1, 120, 16), ([600, 3], [900, 4000], 8, 4, 96, 64), ([2], [20_000], 7, 1, 128, 128), ([1000], [30], 4, 4, 64, 64),
]


@pytest.mark.parametrize("case", range(len(ATTEND_CASES)))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("held,key", [("mx4", "bf16"), ("mx4", "f16"), ("bf16", "bf16"), ("f16", "f16")])
def test_attention_cached(gpu_lib, case, causal, held, key):
    new, lengths, hq, hkv, d, page = ATTEND_CASES[case]
    print(f"[attention] {case} causal={causal} held {held} {key}", flush=True)
    cache, table = make_cache(gpu_lib, lengths, page, hkv, d, held, case)
    q = gen(case)(sum(new), hq, d).to(dtype(key))
    b = ref.offsets_of(new)
    out = gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints(b), causal=causal)
    o, slack = sr.attention_cached(q, cache, table, lengths, b, causal, d ** -0.5)
    ref.check(out, o, slack, "attention")


@pytest.mark.parametrize("held", ["mx4", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_cached_is_attention(gpu_lib, held, rows):
    """The cache's rows gathered and given to the packed attention."""
    import torch
    lengths, new = [300, 1, 77], [rows, 1, 2]
    cache, table = make_cache(gpu_lib, lengths, 32, 2, 64, held, 4)
    q = gen(1)(sum(new), 8, 64).bfloat16()
    kb = ints(ref.offsets_of(lengths))
    k, v = gpu_lib.kv_gather(cache, table, ints(lengths), offsets=kb, n=sum(lengths), out_dtype=torch.bfloat16)
    want = gpu_lib.attention(q, k, v, q_offsets=ints(ref.offsets_of(new)), k_offsets=kb, causal=True).double()
    got = gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints(ref.offsets_of(new))).double()
    # (both round P and the output: twice what either may be off)
    _, slack = sr.attention_cached(q, cache, table, lengths, ref.offsets_of(new), True, 0.125)
    assert bool(((got - want).abs() <= 2 * (slack + 2.0 ** -9 * (want.abs() + slack)) + 1e-30).all())


@pytest.mark.parametrize("held,key", [("mx4", "bf16"), ("mx4", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("rows,hq", [(1, 2), (5, 4), (20, 2), (150, 4)])
def test_attention_cached_behind_the_mask(gpu_lib, held, key, rows, hq):
    """NaN in keys and values that some rows, or none, see; pages that are not the pool's; slots behind the length."""
    import torch
    lengths = [200, 90]
    cache, table = make_cache(gpu_lib, lengths, 16, 2, 64, held, 6)
    # the last slots' rows, which only the last queries see, hold NaN; so do all slots behind the lengths
    bad = torch.full((260, 2, 64), math.nan, device="cuda").to(dtype(key))
    gpu_lib.kv_append(cache, bad[:8], bad[:8], table[:1].contiguous(), ints([208]))       # keys 200..207: one page's end
    ones = gen(2)(2, 2, 64).to(dtype(key))
    nan_v = ones.clone()
    nan_v[1, 0, 5] = math.nan
    gpu_lib.kv_append(cache, ones, nan_v, table[:1].contiguous(), ints([199]))            # value 198 of sample 0
    nan_k = ones.clone()
    nan_k[0, 1, 40] = math.inf
    gpu_lib.kv_append(cache, nan_k, ones, table[1:].contiguous(), ints([89]))             # key 87 of sample 1
    table[0, 3], table[1, 0] = 1 << 20, -1                                                # keys 48..63, 0..15
    q = gen(3)(2 * rows, hq, 64).to(dtype(key))
    b = [0, rows, 2 * rows]
    for causal in (True, False):
        out = gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints(b), causal=causal)
        o, slack = sr.attention_cached(q, cache, table, lengths, b, causal, 0.125)
        ref.check(out, o, torch.nan_to_num(slack), "behind the mask")


@pytest.mark.parametrize("key", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [4, 12, 150])
def test_attention_cached_largest_values(gpu_lib, rows, key):
    """A value at the end of the heads' range, whose code and power are past it, has no effect on the rows that do not see its key."""
    import torch
    cache = gpu_lib.kv_cache(20, 16, 1, 64)
    n = 200
    table = torch.arange(20, dtype=torch.int32, device="cuda").view(1, 20)
    k, v = gen(1)(n, 1, 64).to(dtype(key)), gen(2)(n, 1, 64).to(dtype(key))
    gpu_lib.kv_append(cache, k, v, table, ints([n]))
    q = gen(3)(rows, 2, 64).to(dtype(key))
    want = gpu_lib.attention_cached(q, cache, table, ints([n]))
    v[n - 1, 0, 7] = torch.finfo(dtype(key)).max
    gpu_lib.kv_append(cache, k, v, table, ints([n]))
    got = gpu_lib.attention_cached(q, cache, table, ints([n]))
    assert torch.equal(got[:-1], want[:-1])
    assert bool(torch.isinf(got[-1, :, 7]).all())      # (the code nearest to it stands for 2^128, or 2^16)


def test_attention_cached_falling_offsets(gpu_lib):
    """Offsets that fall give no sample any rows, however many their samples would have together."""
    import torch
    cache, table = make_cache(gpu_lib, [64], 16, 2, 64, "mx4", 8)
    for n in (12, 5000):
        q = gen(4)(n, 4, 64).bfloat16()
        for samples in (3, 64, 301):
            out = torch.full_like(q, 7.0)
            gpu_lib.attention_cached(q, cache, table.expand(samples, -1).contiguous(), ints([64] * samples),
                                     offsets=ints([(i % 2) * n for i in range(samples + 1)]), out=out)
            assert bool((out == 7).all())


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_cached_many_samples(gpu_lib, rows):
    """More samples than a wave has lanes, some empty, in both kernels."""
    import torch
    lengths = [(i * 53) % 190 for i in range(150)]
    cache, table = make_cache(gpu_lib, lengths, 32, 2, 64, "mx4", 3)
    new = [0 if i % 11 == 3 else rows for i in range(150)]
    b = ref.offsets_of(new)
    q = gen(5)(sum(new), 4, 64).bfloat16()
    out = gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints(b))
    o, slack = sr.attention_cached(q, cache, table, lengths, b, True, 0.125)
    ref.check(out, o, slack, "many samples")


@pytest.mark.parametrize("rows", [1, 5, 70])
def test_attention_cached_wide_table(gpu_lib, rows):
    """A table for a billion keys a sample of which few are there: work is counted in coarser steps; the same bits or, where
    the cuts lie elsewhere, within what the cuts allow."""
    import torch
    lengths = [500, 3000]
    cache, table = make_cache(gpu_lib, lengths, 256, 32, 32, "mx4", 3)
    wide = torch.full((2, 1 << 22), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    q = gen(5)(2 * rows, 32, 32).bfloat16()
    b = [0, rows, 2 * rows]
    out = gpu_lib.attention_cached(q, cache, wide, ints(lengths), offsets=ints(b))
    o, slack = sr.attention_cached(q, cache, table, lengths, b, True, 32 ** -0.5)
    ref.check(out, o, slack, "wide table")
    k, _ = gpu_lib.kv_gather(cache, wide, ints(lengths), offsets=ints(b), n=2 * rows)
    assert torch.equal(k, gpu_lib.kv_gather(cache, table, ints(lengths), offsets=ints(b), n=2 * rows)[0])


@pytest.mark.parametrize("held", ["mx4", "bf16"])
def test_attention_cached_skewed(gpu_lib, held):
    """One sample with nearly all keys, or nearly all rows, among many."""
    for new, lengths in (([1] * 9, [3, 4, 20_000, 1, 0, 9, 70, 2, 5]), ([1, 1, 300, 1], [50, 2, 400, 900]), ([1] * 40 + [100], [30] * 41)):
        cache, table = make_cache(gpu_lib, lengths, 64, 2, 128, held, 3)
        b = ref.offsets_of(new)
        q = gen(5)(sum(new), 8, 128).bfloat16()
        out = gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints(b))
        o, slack = sr.attention_cached(q, cache, table, lengths, b, True, 128 ** -0.5)
        ref.check(out, o, slack, f"skewed {len(new)}")


@pytest.mark.parametrize("new,lengths", [([1], [9000]), ([1, 1, 1], [300, 0, 4000]), ([5], [2000]), ([40, 3], [20, 3000]), ([200, 90], [3000, 60])])
@pytest.mark.parametrize("held", ["mx4", "bf16"])
def test_attention_cached_workspace(gpu_lib, new, lengths, held):
    """What the workspace held has no effect; rows that see no key among the cut ones."""
    import torch
    cache, table = make_cache(gpu_lib, lengths, 32, 2, 96, held, 4)
    b = ints(ref.offsets_of(new))
    q = gen(6)(sum(new), 8, 96).bfloat16()
    ws = gpu_lib.attention_cached_workspace(sum(new), len(new), 8, cache, table.shape[1])
    outs = [gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=b, workspace=ws.fill_(v)) for v in (0, 255, 127, 1)]
    o, slack = sr.attention_cached(q, cache, table, lengths, ref.offsets_of(new), True, 96 ** -0.5)
    ref.check(outs[0], o, slack, "workspace")
    assert all(same(outs[0], x) for x in outs[1:])


def test_attention_cached_rows(gpu_lib):
    """Rows of no sample left as they were; lengths past the table and below zero; samples on the same pages; empty caches."""
    import torch
    cache, table = make_cache(gpu_lib, [64, 48], 16, 2, 64, "mx4", 8)
    q = gen(4)(12, 4, 64).bfloat16()
    for lengths in ([64, 48], [1000, -7], [0, 1]):
        out = torch.full_like(q, 7.0)
        gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints([2, 6, 9]), out=out)
        o, slack = sr.attention_cached(q, cache, table, lengths, [2, 6, 9], True, 0.125)
        assert bool((out[:2] == 7).all() and (out[9:] == 7).all())
        ref.check(out[2:9], o[2:9], slack[2:9], f"lengths {lengths}")
    shared = table[[0, 0]].contiguous()
    out = gpu_lib.attention_cached(q[[0, 0]].contiguous(), cache, shared, ints([64, 64]), offsets=ints([0, 1, 2]))
    assert torch.equal(out[0], out[1])
    none = gpu_lib.kv_cache(0, 16, 2, 64)
    out = gpu_lib.attention_cached(q, none, ints([[0, 1]]), ints([20]))
    assert bool((out == 0).all())
    gpu_lib.attention_cached(q, cache, table, ints([64, 48]), offsets=ints([9, -4, 1 << 30]))
    assert gpu_lib.attention_cached(q[:0], cache, table, ints([64, 48]), offsets=ints([0, 0, 0])).shape == (0, 4, 64)
    wide = torch.zeros(12, 6, 64, dtype=torch.bfloat16, device="cuda")      # strided heads, q and out
    wide[:, 1:5] = q
    out = torch.zeros_like(wide)
    got = gpu_lib.attention_cached(wide[:, 1:5], cache, table, ints([64, 48]), offsets=ints([0, 6, 12]), out=out[:, :4])
    assert torch.equal(got, gpu_lib.attention_cached(q, cache, table, ints([64, 48]), offsets=ints([0, 6, 12])))
    assert bool((out[:, 4:] == 0).all())


@pytest.mark.parametrize("spread", [30.0, 3000.0])
@pytest.mark.parametrize("key", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 200])
def test_attention_cached_large_scores(gpu_lib, spread, key, rows):
    """A maximum that grows from tile to tile, scores far from zero: one key takes nearly all."""
    import torch
    cache = gpu_lib.kv_cache(40, 16, 1, 64, dtype(key))
    n = 640
    k = torch.zeros(n, 1, 64, device="cuda")
    k[:, 0, 0] = torch.linspace(-1, 1, n, device="cuda") * spread
    k[:, 0, 1:] = gen(1)(n, 63) * 0.1
    v = gen(2)(n, 1, 64)
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
    gpu_lib.kv_append(cache, k.to(dtype(key)), v.to(dtype(key)), table, ints([n]))
    q = gen(3)(rows, 2, 64).to(dtype(key))
    q[:, :, 0] = 4.0
    out = gpu_lib.attention_cached(q, cache, table, ints([n]), causal=False)
    o, slack = sr.attention_cached(q, cache, table, [n], [0, rows], False, 0.125)
    # (a score of size x is off by d 2^-24 of the sum of its products' sizes, and so is the exponent)
    size = (q.double().abs() @ k[:, 0].to(dtype(key)).double().abs().t()).amax(-1, keepdim=True) * 0.125 * 2.0 ** -18
    ref.check(out, o, slack + size * v.abs().max().item(), "large scores")


# ---- streams, graphs, a run of them ---------------------------------------------------------------
def run_block(pkg, s, qo=None, **kw):
    """A step: norm to 8 bits, the product to q, k and v, the cache, attention to it, the product back to the stream."""
    import torch
    (h, stream), n = pkg.rms_norm(s["x"], s["gamma"], residual=s["r"], out_dtype=torch.float8_e4m3fn, **kw), s["x"].shape[0]
    qkv = pkg.linear_mx(h, s["w_in"], s["b_in"], out_dtype=torch.bfloat16, **kw).view(n, 8, 64)
    q = pkg.kv_append(s["cache"], qkv[:, 4:6], qkv[:, 6:], s["table"], s["lengths"], offsets=s["offsets"], q=qkv[:, :4], pos=s["pos"], **kw)
    o = pkg.attention_cached(q, s["cache"], s["table"], s["lengths"], offsets=s["offsets"], **kw)
    mo = pkg.mx_quantize(o.view(n, 256), **kw)
    return pkg.linear_mx(mo, s["w_out"], residual=stream, out_dtype=torch.float32, **kw)


def block_state(pkg, new, lengths, seed=0):
    import torch
    randn, n = gen(seed), sum(new)
    cache, table = make_cache(pkg, lengths, 32, 2, 64, "mx4", seed)
    return {"x": randn(n, 256).bfloat16(), "r": randn(n, 256), "gamma": 1 + 0.1 * randn(256), "w_in": pkg.mx_quantize(randn(512, 256) / 16),
            "b_in": 0.1 * randn(512), "w_out": pkg.mx_quantize(randn(256, 256) / 16), "cache": cache, "table": table,
            "lengths": ints(lengths), "offsets": ints(ref.offsets_of(new)),
            "pos": torch.cat([torch.arange(e - m, e, dtype=torch.int32) for m, e in zip(new, lengths)])[:, None].cuda()}


@pytest.mark.parametrize("new,lengths", [([1, 1, 1], [90, 33, 1]), ([200, 5], [200, 400])])
def test_block(gpu_lib, new, lengths):
    """Against the same step in 64 bits, each rounding in its place."""
    import torch
    s = block_state(gpu_lib, new, lengths)
    b = ref.offsets_of(new)
    y, h = sr.rms_norm(s["x"], s["r"], s["gamma"], 1e-6)
    out = run_block(gpu_lib, s)
    mx, stream = gpu_lib.rms_norm(s["x"], s["gamma"], residual=s["r"], out_dtype=torch.float8_e4m3fn)
    check_mx(mx, y, "norm")
    z, sl = sr.linear(sr.of_mx(mx), sr.of_mx(s["w_in"]), s["b_in"], "none", None, False)
    qkv = gpu_lib.linear_mx(mx, s["w_in"], s["b_in"])
    ref.check(qkv, z, sl, "qkv")
    qkv = qkv.view(-1, 8, 64)
    yq, sq = ref.rope(qkv[:, :4], s["pos"], [32], 10000.0, True, None, 1e-6)
    q = gpu_lib.kv_append(s["cache"], qkv[:, 4:6], qkv[:, 6:], s["table"], s["lengths"], offsets=s["offsets"], q=qkv[:, :4], pos=s["pos"])
    ref.check(q, yq, sq, "q")
    o, so = sr.attention_cached(q, s["cache"], s["table"], lengths, b, True, 0.125)
    a = gpu_lib.attention_cached(q, s["cache"], s["table"], s["lengths"], offsets=s["offsets"])
    ref.check(a, o, so, "attention")
    ao = gpu_lib.mx_quantize(a.view(-1, 256))
    z, sl = sr.linear(sr.of_mx(ao), sr.of_mx(s["w_out"]), None, "none", stream, True)
    ref.check(out, z, sl, "step")


def test_captured_and_replayed(gpu_lib):
    """A step captured into a graph and replayed as the samples grow, with eager work between the replays."""
    import torch
    new, lengths = [1, 1, 1], [90, 33, 1]
    eager, graphed = block_state(gpu_lib, new, lengths), block_state(gpu_lib, new, lengths)
    for t in range(2):
        warm = torch.cuda.Stream()
        warm.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(warm):
            run_block(gpu_lib, graphed)
        torch.cuda.current_stream().wait_stream(warm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run_block(gpu_lib, graphed)
    for step in range(4):
        for s in (eager, graphed):
            s["x"].copy_(gen(100 + step)(3, 256))
            s["lengths"].copy_(ints([min(m + step, 96 if i == 0 else 64 if i == 1 else 32) for i, m in enumerate(lengths)]))
            s["pos"].copy_((s["lengths"] - 1)[:, None])
        want = run_block(gpu_lib, eager)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {step}"
        assert same(eager["cache"].data, graphed["cache"].data)


def test_other_stream(gpu_lib):
    import torch
    a, b = block_state(gpu_lib, [2, 300], [64, 300]), block_state(gpu_lib, [2, 300], [64, 300])
    want = run_block(gpu_lib, a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = run_block(gpu_lib, b, stream=side)
    side.synchronize()
    assert torch.equal(got, want)


def test_two_calls_at_once(gpu_lib):
    """Calls on two streams with a workspace each, many times over the same inputs: the same bits."""
    import torch
    cache, table = make_cache(gpu_lib, [3000, 20, 700], 64, 2, 128, "mx4", 1)
    q = gen(1)(3, 16, 128).bfloat16()
    args = (cache, table, ints([3000, 20, 700]))
    want = gpu_lib.attention_cached(q, *args, offsets=ints([0, 1, 2, 3]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(10):
        outs.append(gpu_lib.attention_cached(q, *args, offsets=ints([0, 1, 2, 3]), stream=streams[i % 2]))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_rows_past_32_bits(gpu_lib):
    """Norms and linears of more than 4 GiB: the last rows as by themselves."""
    import torch
    n, c = 2_200_003, 1024
    x = torch.zeros((n, c), dtype=torch.bfloat16, device="cuda")
    x[-300:] = gen(1)(300, c).bfloat16()
    tail = x[-300:].clone()
    assert torch.equal(gpu_lib.rms_norm(x)[-300:], gpu_lib.rms_norm(tail))
    m, t = gpu_lib.mx_quantize(x), gpu_lib.mx_quantize(tail)
    assert same(m.codes[-300:], t.codes) and same(m.powers[-300:], t.powers)
    w = gpu_lib.mx_quantize(gen(2)(1000, c) / 32)
    y = gpu_lib.linear_mx(m, w)
    assert y.numel() > 1 << 31 and torch.equal(y[-300:], gpu_lib.linear_mx(t, w))


def test_cache_past_32_bits(gpu_lib):
    """A pool of more than 4 GiB, its last pages in use."""
    import torch
    page_bytes = gpu_lib.lib().tsp_kv_page_bytes(256, 8, 128, gpu_lib.TSP_KV_MX4)
    pages = (5 << 30) // page_bytes
    cache = gpu_lib.KVCache(torch.empty((pages, page_bytes), dtype=torch.uint8, device="cuda"), 256, 8, 128, "mx4")
    small = gpu_lib.kv_cache(3, 256, 8, 128)
    far, near = ints([[pages - 1, 0, pages - 2]]), ints([[2, 0, 1]])
    k, v, q = (gen(i)(600, 8, 128).bfloat16() for i in range(3))
    for c, t in ((cache, far), (small, near)):
        gpu_lib.kv_append(c, k, v, t, ints([600]))
    for rows in (1, 600):
        a = gpu_lib.attention_cached(q[:rows], cache, far, ints([600]))
        assert torch.equal(a, gpu_lib.attention_cached(q[:rows], small, near, ints([600])))
    a, b = gpu_lib.kv_gather(cache, far, ints([600]), n=600), gpu_lib.kv_gather(small, near, ints([600]), n=600)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
