"""Measured operators of a served transformer block, through the package's entry points, over the sizes
it meets.

A model that answers step by step, or samples many steps against the same conditions, keeps the keys and
values of what it has seen in a paged cache and its weights in 8 bits:

  rms_norm  root-mean-square norm of a row with the residual's addition, out in 8 bits with a scale for
            every 32 channels (the next product's operand) or in 16
  linear    x W^T + bias of such 8-bit operands, with SiLU or the residual in its end
  append    new keys and values into a paged cache, the queries and keys RMS-normalised and turned to
            their positions on the way; the cache holds them in 4 bits with a scale for every 32 channels,
            or in 16. A 4-bit cache's new rows are read back in 16 bits, a 16-bit cache is returned as it is
  attend    softmax attention of new queries to a sample's 4-bit or 16-bit cache: single tokens, drafts of
            a few, pieces of a prompt, and conditions that every row sees whole

8 bits: e4m3 codes and one power of two (e8m0) for 32 channels, the least one with which the largest of
them is at most 448. 4 bits: e2m1 codes, the same with 6; element 2i in a byte's low half. A page holds
`page` tokens of every key head: for each head the K codes [page][16 B], the V codes alike, K's
powers [page][B] and V's, B = ceil(d / 32); in 16 bits K [page][d] and V alike.

Samples are ragged: a batch of three or more holds one of a single row, of five or more an empty one.
Features are standard normal, the residual stream is wider.
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "mx8": 1 + 1 / 32}
THETA = 10000.0
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# the largest listed cases: products of a linear and its outputs, bytes of a norm, score pairs times
# channels of an attention
MOST_LINEAR, MOST_OUTPUTS = 35_001 * 4_096 * 1_024, 35_001 * 1_024
MOST_NORM = 60_013 * 2_048 * 8
MOST_ATTEND = 200_000_000_000


def _package():
    """The package directory's name holds a dot, so it is loaded by path."""
    if "trellis_cpp_amd" not in sys.modules:
        pkg_dir = os.path.join(ROOT, "trellis.cpp_amd")
        spec = importlib.util.spec_from_file_location("trellis_cpp_amd", os.path.join(pkg_dir, "__init__.py"),
                                                      submodule_search_locations=[pkg_dir])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["trellis_cpp_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["trellis_cpp_amd"]


# ---- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # one new token of each of five samples: launches count
        {"name": "norm_5_c1024", "op": "rms_norm", "n": 5, "c": 1024, "dtype": "bf16", "residual": "bf16", "out": "mx8"},
        # a 64^3 level's rows at 1024 channels, an f32 residual stream, into the next product's 8 bits
        {"name": "norm_35k_c1024", "op": "rms_norm", "n": 35_001, "c": 1024, "dtype": "bf16", "residual": "f32", "out": "mx8"},
        # a large batch of wide rows that stay in 16 bits
        {"name": "norm_60k_c2048", "op": "rms_norm", "n": 60_013, "c": 2048, "dtype": "bf16", "residual": "bf16", "out": "bf16"},
        # the first product of a step's MLP for five tokens: the weights are all there is to read
        {"name": "linear_5_c4096", "op": "linear", "n": 5, "ci": 1024, "co": 4096, "act": "silu", "bias": True, "residual": False,
         "out": "bf16"},
        # a small object's rows, an odd number of outputs
        {"name": "linear_2k_c1000", "op": "linear", "n": 2_606, "ci": 1024, "co": 1000, "act": "none", "bias": True,
         "residual": False, "out": "f16"},
        # the second product of an MLP over a 64^3 level, added to the residual stream
        {"name": "linear_35k_c1024", "op": "linear", "n": 35_001, "ci": 4096, "co": 1024, "act": "none", "bias": True,
         "residual": True, "out": "f32"},
        # one new token of each of 16 samples into their caches
        {"name": "append_16_mx4", "op": "append", "n": 16, "samples": 16, "before": 8_000, "hq": 16, "hkv": 4, "d": 128, "page": 64,
         "axes": 1, "interleaved": False, "norm": True, "dtype": "bf16", "held": "mx4"},
        # a packed batch of prompts, four heads of q on one of k and v
        {"name": "append_12k_mx4", "op": "append", "n": 12_345, "samples": 7, "before": 100, "hq": 16, "hkv": 4, "d": 128, "page": 64,
         "axes": 1, "interleaved": False, "norm": True, "dtype": "bf16", "held": "mx4"},
        # voxels at their places on three axes into a cache of 16 bits
        {"name": "append_60k_16", "op": "append", "n": 60_013, "samples": 2, "before": 0, "hq": 16, "hkv": 16, "d": 64, "page": 256,
         "axes": 3, "interleaved": True, "norm": False, "dtype": "f16", "held": "16"},
        # one new token against a long cache, eight heads of q on one of k and v
        {"name": "attend_1_in_40k", "op": "attend", "nq": 1, "nk": 40_009, "samples": 1, "hq": 16, "hkv": 2, "d": 128, "page": 64,
         "causal": True, "dtype": "bf16", "held": "mx4"},
        # a batch of 16 samples' new tokens against their caches, of unequal length
        {"name": "attend_16_in_400k", "op": "attend", "nq": 16, "nk": 400_009, "samples": 16, "hq": 16, "hkv": 4, "d": 128, "page": 64,
         "causal": True, "dtype": "bf16", "held": "mx4"},
        # pieces of two prompts behind what their caches hold already
        {"name": "attend_5k_in_35k", "op": "attend", "nq": 5_003, "nk": 35_001, "samples": 2, "hq": 16, "hkv": 4, "d": 128, "page": 64,
         "causal": True, "dtype": "bf16", "held": "mx4"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))


def draw(rng):
    op = rng.choice(["rms_norm", "rms_norm", "linear", "linear", "append", "append", "attend", "attend", "attend", "attend"])
    if op == "rms_norm":
        c = rng.choice([64, 96, 128, 320, 500, 512, 768, 1000, 1024, 1536, 2048, 4096, 5120, 8192])
        dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
        residual = rng.choice(["none", "f32", dtype, dtype])
        out = rng.choice(["mx8", "mx8", "bf16", "f16"]) if c % 32 == 0 else "bf16"
        each = SIZE[dtype] + SIZE[out] + 2 * (0 if residual == "none" else SIZE[residual])
        return {"op": op, "n": _log_int(rng, 1, int(MOST_NORM / each) // c), "c": c, "dtype": dtype, "residual": residual, "out": out}
    if op == "linear":
        ci = rng.choice([96, 128, 160, 256, 512, 768, 1024, 1536, 2048, 4096, 8192])
        co = rng.choice([27, 64, 100, 256, 333, 512, 768, 1000, 1024, 2048, 4096, 8192])
        act = rng.choice(["none", "silu"])
        return {"op": op, "n": _log_int(rng, 1, min(120_000, MOST_LINEAR // (ci * co), MOST_OUTPUTS // co)), "ci": ci, "co": co, "act": act,
                "bias": rng.random() < 0.7, "residual": act == "none" and rng.random() < 0.5,
                "out": rng.choice(["f32", "f16", "bf16", "bf16"])}
    d = rng.choice([32, 64, 80, 96, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    share = rng.choice([1, 2, 4, 8])
    page, held = rng.choice([16, 32, 64, 128, 256]), rng.choice(["mx4", "mx4", "mx4", "16"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "append":
        hq = hkv * share
        return {"op": op, "n": _log_int(rng, 1, 120_000_000 // ((hq + 2 * hkv) * d)), "samples": rng.choice([1, 2, 5, 16]),
                "before": _log_int(rng, 1, 2_000), "hq": hq, "hkv": hkv, "d": d, "page": page, "axes": rng.choice([1, 1, 2, 3]),
                "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5, "dtype": dtype, "held": held}
    hq = min(hkv * share, 16)
    form = rng.choice(["step", "step", "draft", "piece", "condition"])
    samples = rng.choice([1, 2, 5, 16, 40])
    nk = _log_int(rng, 2 * samples, 1_000_000 // hkv)
    most = max(1, MOST_ATTEND // (nk * hq * d))
    if form == "step":
        nq = samples
    elif form == "draft":
        nq = samples * rng.choice([2, 3, 5, 8])
    else:
        samples = rng.choice([1, 1, 2, 5])
        nq = _log_int(rng, 1, min(60_000, most))
        if form == "piece":
            nq = min(nq, nk)
    return {"op": op, "nq": nq, "nk": nk, "samples": samples, "hq": hq, "hkv": hkv, "d": d, "page": page,
            "causal": form != "condition", "dtype": dtype, "held": held}


def _lengths(n, samples):
    """n rows over the samples: one of a single row among three or more, an empty one among five or
    more, the others of unequal size."""
    fixed = {}
    if samples >= 3:
        fixed[1] = 1
    if samples >= 5:
        fixed[3] = 0
    rest = [i for i in range(samples) if i not in fixed]
    left = max(0, n - sum(fixed.values()))
    weights = [3 + (5 * i) % 7 for i in range(len(rest))]
    sizes = [left * w // sum(weights) for w in weights]
    sizes[-1] += left - sum(sizes)
    out = [min(fixed.get(i, 0), n) for i in range(samples)]
    for i, s in zip(rest, sizes):
        out[i] = s
    return out


def _offsets(lengths):
    out = [0]
    for m in lengths:
        out.append(out[-1] + m)
    return out


def _new_rows(n, samples):
    """New rows of each sample: the same few of all where they divide so, else ragged."""
    if n % samples == 0 and n // samples <= 8:
        return [n // samples] * samples
    return _lengths(n, samples)


def _shape(case):
    """(new rows of each sample, keys of each sample after them, pages of each, pages in the pool)"""
    if case["op"] == "append":
        new = _new_rows(case["n"], case["samples"])
        keys = [(case["before"] * (1 + i % 3)) // 2 + m for i, m in enumerate(new)]
    else:
        new, keys = _new_rows(case["nq"], case["samples"]), _lengths(case["nk"], case["samples"])
    pages = [-(-m // case["page"]) for m in keys]
    return new, keys, pages, sum(pages) + 3


def _blocks(case):
    return -(-case["d"] // 32)


def _head_bytes(case):
    """Bytes of one key head in one page."""
    return case["page"] * (34 * _blocks(case) if case["held"] == "mx4" else 4 * case["d"])


def _pairs(case):
    return [case["d"] // 2 // case["axes"]] * case["axes"]


# ---- numbers of few bits ----------------------------------------------------------------------
def _power(amax, most):
    """The e8m0 code of the least power of two with which amax is at most `most` = (1 + f) 2^p."""
    near = amax.float()                 # rounded up, which leaves it on its side of every power
    near = torch.where(near < amax, torch.nextafter(near, torch.full_like(near, math.inf)), near)
    bits = near.view(torch.int32)
    f, p = {448: (0x600000, 8), 6: (0x400000, 2)}[most]
    return (((bits + (0x7FFFFF - f)) >> 23) - p).clamp_(min=0).to(torch.uint8)


def _scale(code):
    """2^(code - 127) in 32 bits."""
    return torch.ldexp(torch.ones((), device=code.device), code.to(torch.int32) - 127)


def _blocked(x, block=32):
    """x [..., c] as [..., blocks, 32], zeros behind its last channel."""
    c = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -c % block)).unflatten(-1, (-1, block))


def _to_mx8(x):
    """x f32 [..., c] -> (e4m3 codes [..., c], e8m0 codes [..., c / 32])"""
    b = _blocked(x)
    code = _power(b.abs().amax(-1), 448)
    return (b / _scale(code)[..., None]).flatten(-2).to(torch.float8_e4m3fn), code


def _to_mx4(x):
    """x f32 or f64 [..., d] -> (e2m1 codes [..., blocks, 32] with the sign in bit 3, e8m0 codes [..., blocks])"""
    b = _blocked(x)
    code = _power(b.abs().amax(-1), 6)
    y = b / _scale(code)[..., None]
    a = y.abs()
    # halfway between two values the one with an even code
    mag = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    return mag.byte() | (torch.signbit(y).byte() << 3), code


def _of_mx4(codes, power, d):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    return (table[codes.long()] * _scale(power)[..., None]).flatten(-2)[..., :d]


# ---- the cache --------------------------------------------------------------------------------
def _parts(cache, case):
    """A 4-bit cache's K codes, V codes [pages, heads, page, 16 B], K powers, V powers [..., B]; a 16-bit
    one's K and V [pages, heads, page, d]."""
    h, p, b = case["hkv"], case["page"], _blocks(case)
    heads = cache.view(cache.shape[0], h, -1)
    if case["held"] != "mx4":
        kv = heads.view(DTYPES[case["dtype"]]).view(cache.shape[0], h, 2, p, case["d"])
        return kv[:, :, 0], kv[:, :, 1]
    ends = [16 * b * p, 32 * b * p, 33 * b * p, 34 * b * p]
    return tuple(heads[:, :, a:e].unflatten(2, (p, -1)) for a, e in zip([0] + ends, ends))


def _write(cache, case, page, slot, k, v):
    """Rows k, v [n, heads, d] (f32 or f64) at page[i], slot[i]."""
    parts = _parts(cache, case)
    if case["held"] != "mx4":
        parts[0][page, :, slot] = k.to(parts[0].dtype)
        parts[1][page, :, slot] = v.to(parts[1].dtype)
        return
    for i, x in enumerate((k, v)):
        codes, power = _to_mx4(x)
        codes = codes.flatten(-2)
        parts[i][page, :, slot] = codes[..., 0::2] | (codes[..., 1::2] << 4)
        parts[2 + i][page, :, slot] = power


def _read(cache, case, page, slot):
    """K and V [n, heads, d] (f32) of rows at page[i], slot[i]."""
    parts = _parts(cache, case)
    if case["held"] != "mx4":
        return parts[0][page, :, slot].float(), parts[1][page, :, slot].float()
    out = []
    for i in range(2):
        b = parts[i][page, :, slot]
        codes = torch.stack([b & 15, b >> 4], -1).flatten(-2).unflatten(-1, (-1, 32))
        out.append(_of_mx4(codes, parts[2 + i][page, :, slot], case["d"]))
    return out


# ---- inputs -----------------------------------------------------------------------------------
def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    if case["op"] == "rms_norm":
        n, c = case["n"], case["c"]
        s = {"x": randn(n, c).to(DTYPES[case["dtype"]]), "gamma": 1 + 0.2 * randn(c), "residual": None}
        if case["residual"] != "none":
            s["residual"] = randn(n, c).mul_(4).to(DTYPES[case["residual"]])
        return s
    if case["op"] == "linear":
        n, ci, co = case["n"], case["ci"], case["co"]
        s = {"x": _to_mx8(randn(n, ci)), "w": _to_mx8(randn(co, ci) / math.sqrt(ci)), "bias": None, "residual": None}
        if case["bias"]:
            s["bias"] = 0.2 * randn(co)
        if case["residual"]:
            s["residual"] = randn(n, co)
        return s
    hq, hkv, d, dt = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    new, keys, pages, pool = _shape(case)
    n = sum(new)
    order = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)     # which pages are whose
    table = torch.full((len(pages), max(1, max(pages))), -1, dtype=torch.int32, device=dev)
    for i, (a, m) in enumerate(zip(_offsets(pages), pages)):
        table[i, :m] = order[a: a + m]
    s = {"new": new, "keys": keys, "table": table, "offsets": torch.tensor(_offsets(new), dtype=torch.int32, device=dev),
         "lengths": torch.tensor(keys, dtype=torch.int32, device=dev), "q": randn(n, hq, d).to(dt)}
    cache = torch.zeros((pool, hkv * _head_bytes(case)), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 25) // (hkv * d * case["page"]))
    slots = torch.arange(case["page"], device=dev)
    for a in range(0, pool, step):
        m = min(step, pool - a)
        k, v = randn(2, m * case["page"], hkv, d)
        _write(cache, case, torch.arange(a, a + m, device=dev).repeat_interleave(case["page"]), slots.repeat(m), k, v)
    s["cache"] = cache
    if case["op"] == "append":
        s["k"], s["v"] = randn(n, hkv, d).to(dt), randn(n, hkv, d).to(dt)
        s["q_gamma"] = s["k_gamma"] = None
        if case["norm"]:
            s["q_gamma"], s["k_gamma"] = 1 + 0.2 * randn(hq, d), 1 + 0.2 * randn(hkv, d)
        if case["axes"] == 1:       # a token's place in its sample
            s["pos"] = torch.cat([torch.arange(e - m, e, dtype=torch.int32) for m, e in zip(new, keys)])[:, None].to(dev)
        else:
            s["pos"] = torch.randint(0, 128, (n, case["axes"]), generator=gen, device=dev, dtype=torch.int32)
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:     # what a program keeps from call to call: output buffers, workspaces, the cache's handle
        pkg = _package()
        dev = torch.device("cuda")
        if case["op"] == "rms_norm":
            n, c = case["n"], case["c"]
            state["result"] = (pkg.mx_empty(n, c, dev) if case["out"] == "mx8"
                               else torch.empty((n, c), dtype=DTYPES[case["out"]], device=dev))
            state["sum"] = None if state["residual"] is None else torch.empty_like(state["residual"])
        elif case["op"] == "linear":
            state["x"], state["w"] = (pkg.Mx(codes, power.view(torch.float8_e8m0fnu)) for codes, power in (state["x"], state["w"]))
            state["result"] = torch.empty((case["n"], case["co"]), dtype=DTYPES[case["out"]], device=dev)
            state["workspace"] = pkg.linear_mx_workspace(case["n"], case["ci"], case["co"], dev)
        else:
            held = "mx4" if case["held"] == "mx4" else DTYPES[case["dtype"]]
            cache = pkg.kv_cache(state["cache"].shape[0], case["page"], case["hkv"], case["d"], held, dev)
            cache.data.copy_(state["cache"])
            state["cache"] = cache
            state["q_result"] = torch.empty_like(state["q"])
            if case["op"] == "append":
                state["k_result"], state["v_result"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])
            else:
                state["workspace"] = pkg.attention_cached_workspace(case["nq"], case["samples"], case["hq"], cache,
                                                                    state["table"].shape[1])
    return state


# ---- one pass ---------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        pkg = _package()
        if case["op"] == "rms_norm":
            return pkg.rms_norm(state["x"], state["gamma"], eps=EPS, residual=state["residual"], residual_out=state["sum"],
                                out=state["result"])
        if case["op"] == "linear":
            return pkg.linear_mx(state["x"], state["w"], state["bias"], act=case["act"], residual=state["residual"],
                                 out=state["result"], workspace=state["workspace"])
        if case["op"] == "attend":
            return pkg.attention_cached(state["q"], state["cache"], state["table"], state["lengths"], offsets=state["offsets"],
                                        causal=case["causal"], out=state["q_result"], workspace=state["workspace"])
        q = pkg.kv_append(state["cache"], state["k"], state["v"], state["table"], state["lengths"], offsets=state["offsets"],
                          q=state["q"], pos=state["pos"], pairs=_pairs(case), theta=THETA, interleaved=case["interleaved"],
                          q_gamma=state["q_gamma"], k_gamma=state["k_gamma"], eps=EPS, q_out=state["q_result"])
        if case["held"] != "mx4":
            return q, state["cache"].data.view(DTYPES[case["dtype"]])
        return q, *pkg.kv_gather(state["cache"], state["table"], state["lengths"], offsets=state["offsets"],
                                 k_out=state["k_result"], v_out=state["v_result"])
    if case["op"] == "rms_norm":
        return _plain_rms_norm(state, case)
    if case["op"] == "linear":
        return _plain_linear(state, case)
    if case["op"] == "append":
        return _plain_append(state, case)
    return _plain_attend(state, case)


def _plain_rms_norm(state, case):
    h = state["x"].float()
    if state["residual"] is not None:
        h = h + state["residual"].float()
    y = h / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + EPS) * state["gamma"]
    if case["out"] == "mx8":
        codes, power = _to_mx8(y)
        y = (codes, power.view(torch.float8_e8m0fnu))
    else:
        y = y.to(DTYPES[case["out"]])
    return y if state["residual"] is None else (y, h.to(state["residual"].dtype))


def _plain_linear(state, case):
    x, w = ((codes.float().unflatten(-1, (-1, 32)) * _scale(power)[..., None]).flatten(-2) for codes, power in (state["x"], state["w"]))
    y = torch.matmul(x, w.t())
    if state["bias"] is not None:
        y = y + state["bias"]
    if case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    if state["residual"] is not None:
        y = y + state["residual"]
    return y.to(DTYPES[case["out"]])


def _places(state, case, rows):
    """The page and the slot in it of each sample's last rows[s] keys."""
    page, slot = [], []
    for i, (m, keys) in enumerate(zip(rows, state["keys"])):
        at = torch.arange(keys - m, keys, device=state["table"].device)
        page.append(state["table"][i, at // case["page"]].long())
        slot.append(at % case["page"])
    return torch.cat(page), torch.cat(slot)


def _plain_append(state, case):
    d = case["d"]
    angles = []
    for a, pairs in enumerate(_pairs(case)):
        exponent = -torch.arange(pairs, device=state["pos"].device, dtype=torch.float64) / pairs
        angles.append(state["pos"][:, a, None].double() * THETA ** exponent)
    angle = torch.cat(angles, dim=1)                   # in 64 bits: a far position's turn needs them
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    turned = angle.shape[1]
    out = []
    for x, gamma in ((state["q"], state["q_gamma"]), (state["k"], state["k_gamma"])):
        y = x.double()                                 # and a key next to the border between two codes
        if gamma is not None:
            y = y / torch.sqrt((y * y).mean(dim=-1, keepdim=True) + EPS) * gamma
        first, second = (y[..., 0::2], y[..., 1::2]) if case["interleaved"] else (y[..., : d // 2], y[..., d // 2:])
        u, w = first[..., :turned], second[..., :turned]
        first = torch.cat([u * cos - w * sin, first[..., turned:]], dim=-1)
        second = torch.cat([w * cos + u * sin, second[..., turned:]], dim=-1)
        y = torch.stack([first, second], dim=-1).flatten(-2) if case["interleaved"] else torch.cat([first, second], dim=-1)
        out.append(y)
    page, slot = _places(state, case, state["new"])
    _write(state["cache"], case, page, slot, out[1], state["v"].float())
    q = out[0].to(state["q"].dtype)
    if case["held"] != "mx4":
        return q, state["cache"].view(DTYPES[case["dtype"]])
    k, v = _read(state["cache"], case, page, slot)
    return q, k.to(q.dtype), v.to(q.dtype)


def _plain_attend(state, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    share = hq // hkv
    out = torch.zeros_like(state["q"])
    page, slot = _places(state, case, state["keys"])
    bounds, key_bounds = _offsets(state["new"]), _offsets(state["keys"])
    for qa, qe, ka, ke in zip(bounds, bounds[1:], key_bounds, key_bounds[1:]):
        nq, nk = qe - qa, ke - ka
        if nq == 0 or nk == 0:
            continue
        k, v = _read(state["cache"], case, page[ka:ke], slot[ka:ke])
        k = k.permute(1, 2, 0).contiguous()                                 # [hkv, d, nk]
        v = v.permute(1, 0, 2).contiguous()                                 # [hkv, nk, d]
        step = max(1, (1 << 28) // (nk * hq))                               # the scores of a step fit 1 GiB
        for a in range(0, nq, step):
            b = min(nq, a + step)
            q = state["q"][qa + a: qa + b].float().reshape(b - a, hkv, share, d).permute(1, 2, 0, 3)
            s = torch.matmul(q.reshape(hkv, share * (b - a), d), k) * (1 / math.sqrt(d))
            if case["causal"]:
                last = torch.arange(a, b, device=s.device) + (nk - nq)
                hidden = torch.arange(nk, device=s.device)[None] > last[:, None]
                s = s.reshape(hkv, share, b - a, nk).masked_fill_(hidden, -math.inf).reshape(hkv, share * (b - a), nk)
            top = s.amax(dim=-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            total = p.sum(dim=-1, keepdim=True)
            o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
            out[qa + a: qa + b] = o.reshape(hkv, share, b - a, d).permute(2, 0, 1, 3).reshape(b - a, hq, d).to(out.dtype)
    return out


# ---- what a pass cannot do without ------------------------------------------------------------
def _visible(case):
    new, keys, _, _ = _shape(case)
    total = 0
    for nq, nk in zip(new, keys):
        if not case["causal"]:
            total += nq * nk
        else:               # row i sees max(0, nk - nq + i + 1) keys
            first, rows = max(0, nk - nq + 1), min(nq, nk)
            total += rows * (first + nk) // 2 if rows else 0
    return total


def work(case):
    if case["op"] == "rms_norm":
        e = case["n"] * case["c"]
        moved = SIZE[case["dtype"]] + SIZE[case["out"]] + 2 * (0 if case["residual"] == "none" else SIZE[case["residual"]])
        return {"bytes": e * moved + 4 * case["c"], "flops": 6 * e}
    if case["op"] == "linear":
        n, ci, co = case["n"], case["ci"], case["co"]
        out = n * co * (SIZE[case["out"]] + (4 if case["residual"] else 0)) + (4 * co if case["bias"] else 0)
        return {"bytes": (n + co) * ci * SIZE["mx8"] + out, "flops": 2 * n * ci * co}
    d, row = case["d"], 2 * (17 * _blocks(case) if case["held"] == "mx4" else 2 * case["d"])
    if case["op"] == "append":
        n, hq, hkv = case["n"], case["hq"], case["hkv"]
        read_back = row + 4 * d if case["held"] == "mx4" else 0
        return {"bytes": n * (4 * hq * d + hkv * (4 * d + row + read_back) + 4 * case["axes"]),
                "flops": (7 if case["norm"] else 3) * n * (hq + hkv) * d}
    return {"bytes": case["nk"] * case["hkv"] * row + 4 * case["nq"] * case["hq"] * d,
            "flops": 4 * d * case["hq"] * _visible(case)}


# ---- the definitions in 64 bits ---------------------------------------------------------------
def _exact_power(amax, most):
    """2^e for the least e with amax <= most 2^e (whole steps: exact)."""
    m, e = torch.frexp(amax / most)         # amax / most = m 2^e, 1/2 <= m < 1
    return torch.ldexp(torch.ones_like(amax), torch.where(m == 0.5, e - 1, e))


def _exact_mx4(x):
    """x [n, h, d] as its 4-bit codes stand for it."""
    n, h, d = x.shape
    y = torch.zeros((n, h, -(-d // 32) * 32), dtype=torch.float64, device=x.device)
    y[..., :d] = x
    y = y.view(n, h, -1, 32)
    power = _exact_power(y.abs().amax(3, keepdim=True), 6)
    y = y / power
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)      # of the values about y: 1/2, 1 or 2
    return (torch.round(y / step) * step * power).reshape(n, h, -1)[..., :d]


def _exact_cache(case, s):
    """K and V of each sample in 64 bits, [keys, heads, d], from the bytes."""
    p, b, h, d = case["page"], _blocks(case), case["hkv"], case["d"]
    values = torch.tensor([(-1) ** (c >> 3) * (E2M1[c & 7]) for c in range(16)], dtype=torch.float64, device=s["cache"].device)
    for i, keys in enumerate(s["keys"]):
        if keys == 0:
            yield None, None
            continue
        pages = s["cache"][s["table"][i, : -(-keys // p)].long()].reshape(-1, h, _head_bytes(case))
        kv = []
        for side in range(2):
            if case["held"] == "mx4":
                codes = pages[..., side * 16 * b * p: (side + 1) * 16 * b * p].reshape(-1, h, p, 16 * b)
                power = pages[..., (32 + side) * b * p: (33 + side) * b * p].reshape(-1, h, p, b)
                x = torch.empty((*codes.shape[:-1], 32 * b), dtype=torch.float64, device=codes.device)
                x[..., 0::2], x[..., 1::2] = values[(codes % 16).long()], values[(codes // 16).long()]
                x *= torch.exp2(power.double() - 127).repeat_interleave(32, dim=-1)
            else:
                x = pages[..., side * 2 * d * p: (side + 1) * 2 * d * p].contiguous().view(DTYPES[case["dtype"]]).reshape(-1, h, p, d).double()
            kv.append(x[..., :d].transpose(1, 2).reshape(-1, h, d)[:keys])
        yield kv[0], kv[1]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rms_norm":
        total = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = total * torch.rsqrt(total.square().mean(1, keepdim=True) + EPS) * s["gamma"].double()
        if case["out"] == "mx8":        # the codes before their rounding
            y = y.view(case["n"], -1, 32)
            y = ((y / _exact_power(y.abs().amax(2, keepdim=True), 448)).reshape(case["n"], -1), None)
        return y if s["residual"] is None else (y, total)
    if case["op"] == "linear":
        x, w = ((codes.double() * torch.exp2(power.double() - 127).repeat_interleave(32, 1)) for codes, power in (s["x"], s["w"]))
        y = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
        if case["act"] == "silu":
            y = y * torch.sigmoid(y)
        return y if s["residual"] is None else y + s["residual"].double()
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        n = s["pos"].shape[0]
        turn = torch.ones((n, d // 2), dtype=torch.complex128, device=s["pos"].device)
        j = 0
        for axis, pairs in enumerate(_pairs(case)):
            for i in range(pairs):
                angle = s["pos"][:, axis].double() * math.pow(THETA, -i / pairs)
                turn[:, j] = torch.polar(torch.ones_like(angle), angle)
                j += 1
        out = []
        for x, gamma in ((s["q"], s["q_gamma"]), (s["k"], s["k_gamma"])):
            heads = []
            for h in range(x.shape[1]):
                y = x[:, h].double()
                if gamma is not None:
                    y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + EPS) * gamma[h].double()
                z = y.reshape(-1, d // 2, 2) if case["interleaved"] else y.reshape(-1, 2, d // 2).transpose(1, 2)
                z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
                heads.append(z.reshape(-1, d) if case["interleaved"] else z.transpose(1, 2).reshape(-1, d))
            out.append(torch.stack(heads, dim=1))
        if case["held"] == "mx4":
            return out[0], _exact_mx4(out[1]), _exact_mx4(s["v"].double())
        cache = s["cache"].view(DTYPES[case["dtype"]]).double()
        pages = cache.view(-1, hkv, 2, case["page"], d)
        row = 0
        for i, (m, keys) in enumerate(zip(s["new"], s["keys"])):
            at = torch.arange(keys - m, keys, device=cache.device)
            page = s["table"][i].long()[torch.div(at, case["page"], rounding_mode="floor")]
            pages[page, :, 0, at % case["page"]] = out[1][row: row + m]
            pages[page, :, 1, at % case["page"]] = s["v"][row: row + m].double()
            row += m
        return out[0], cache
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    row = 0
    for m, keys, (k, v) in zip(s["new"], s["keys"], _exact_cache(case, s)):
        if m and keys:
            step = max(1, (1 << 27) // keys)
            for h in range(hq):
                kh, vh = k[:, h * hkv // hq].contiguous(), v[:, h * hkv // hq].contiguous()
                for a in range(0, m, step):
                    b = min(m, a + step)
                    scores = s["q"][row + a: row + b, h].double() @ kh.t() / math.sqrt(d)
                    if case["causal"]:
                        i = torch.arange(a - m, b - m, device=scores.device)      # counted from the end
                        j = torch.arange(-keys, 0, device=scores.device)
                        scores = scores.masked_fill(j[None] > i[:, None], -math.inf)
                    seen = torch.isfinite(scores).any(dim=1, keepdim=True)
                    p = torch.softmax(torch.where(seen, scores, torch.zeros_like(scores)), dim=1)
                    out[row + a: row + b, h] = torch.where(seen, p @ vh, torch.zeros_like(out[row + a: row + b, h]))
        row += m
    return out
