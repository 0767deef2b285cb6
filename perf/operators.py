"""Measured operators of a voxel transformer's block, through the package's entry points, over the
sizes it meets.

A model over voxels (or over image and video patches) runs, on packed rows of several samples:

  group_norm  group norm over each sample's rows and a group's channels, channels last, with SiLU
  rope        rotary positions on several axes: q and k turned by their integer coordinates, with
              an RMS norm of every head first where the model normalises q and k
  attention   softmax attention within each sample: voxels to themselves, voxels to an image's
              tokens, causal sequences, and one or a few new tokens against a long cache; heads of q
              may share a head of k and v

Samples are ragged: a packed batch of three samples or more holds one of a single row, of five or
more an empty one. Features are standard normal (group norm: with a mean and a spread that differ by
channel, as a conv's output has them).
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
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 10000.0
EPS = 1e-6
# the largest listed attention case: score pairs times channels
MOST = 35_001 * 35_001 * 1024


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
        # a small object's 32^3 latent in a narrow layer: launches count
        {"name": "norm_2k_c64", "op": "group_norm", "n": 2_606, "c": 64, "groups": 32, "samples": 1, "silu": True,
         "dtype": "f32", "out": "f16"},
        # a batch of objects at the third stage's width, 16-bit features in and out
        {"name": "norm_60k_c256", "op": "group_norm", "n": 60_013, "c": 256, "groups": 32, "samples": 6, "silu": True,
         "dtype": "bf16", "out": "bf16"},
        # the last stage at 512^3: the f32 residual stream normalised into the next product's input
        {"name": "norm_600k_c128", "op": "group_norm", "n": 599_577, "c": 128, "groups": 32, "samples": 2, "silu": True,
         "dtype": "f32", "out": "bf16"},
        # the tokens of one step, two axes (an image's rows and columns)
        {"name": "rope_97_h16", "op": "rope", "n": 97, "hq": 16, "hk": 16, "d": 64, "axes": 2, "grid": 64, "interleaved": False,
         "norm": False, "dtype": "f16"},
        # a level of voxels, q and k normalised and turned, in 16 bits
        {"name": "rope_35k_h8", "op": "rope", "n": 35_001, "hq": 8, "hk": 8, "d": 128, "axes": 3, "grid": 64, "interleaved": True,
         "norm": True, "dtype": "bf16"},
        # a larger level with few key heads
        {"name": "rope_117k_h16", "op": "rope", "n": 117_343, "hq": 16, "hk": 4, "d": 64, "axes": 3, "grid": 128,
         "interleaved": True, "norm": True, "dtype": "f16"},
        # one new token against a long cache, eight heads of q on one of k and v
        {"name": "attend_1_in_40k", "op": "attention", "nq": 1, "nk": 40_009, "samples": 1, "hq": 16, "hkv": 2, "d": 128,
         "causal": True, "dtype": "bf16"},
        # a small object's voxels to themselves
        {"name": "attend_2k_h8", "op": "attention", "nq": 2_606, "nk": 2_606, "samples": 1, "hq": 8, "hkv": 8, "d": 64,
         "causal": False, "dtype": "f16"},
        # voxels to the tokens of their image
        {"name": "attend_14k_in_1k", "op": "attention", "nq": 14_487, "nk": 1_029, "samples": 1, "hq": 16, "hkv": 16, "d": 64,
         "causal": False, "dtype": "bf16"},
        # a packed batch of causal sequences of different lengths, four heads of q on one of k and v
        {"name": "attend_packed_12k", "op": "attention", "nq": 12_345, "nk": 12_345, "samples": 7, "hq": 16, "hkv": 4, "d": 128,
         "causal": True, "dtype": "bf16"},
        # a 64^3 level's voxels to themselves at 1024 channels: the largest
        {"name": "attend_35k_h8", "op": "attention", "nq": 35_001, "nk": 35_001, "samples": 1, "hq": 8, "hkv": 8, "d": 128,
         "causal": False, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "rope", "rope", "attention", "attention", "attention", "attention"])
    if op == "group_norm":
        c = rng.choice([32, 64, 96, 128, 192, 256, 320, 512, 640, 1024])
        n = _log_int(rng, 64, 80_000_000 // c)
        dtype = rng.choice(["f32", "f16", "bf16"])
        return {"op": op, "n": n, "c": c, "groups": rng.choice([8, 16, 32]), "samples": rng.choice([1, 1, 2, 5, 16]),
                "silu": rng.random() < 0.75, "dtype": dtype, "out": rng.choice([dtype, "bf16", "f16"])}
    if op == "rope":
        d = rng.choice([32, 64, 80, 96, 128])
        hq = rng.choice([4, 8, 12, 16])
        return {"op": op, "n": _log_int(rng, 1, 150_000_000 // (hq * d)), "hq": hq, "hk": rng.choice([hq, hq, hq // 2, hq // 4]),
                "d": d, "axes": rng.choice([1, 2, 3, 3]), "grid": rng.choice([64, 512, 100_000]),
                "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5, "dtype": rng.choice(["f32", "f16", "bf16"])}
    d = rng.choice([64, 64, 80, 96, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 1, 2, 4]) if hkv > 1 else rng.choice([4, 8])
    dtype = rng.choice(["f16", "bf16"])
    form = rng.choice(["self", "self", "causal", "causal", "cross", "step"])
    if form == "step":          # one or a few new tokens of every sample against its cache
        samples = rng.choice([1, 2, 5, 16])
        return {"op": op, "nq": samples * rng.choice([1, 1, 3, 8]), "nk": _log_int(rng, 512, 400_000), "samples": samples,
                "hq": hq, "hkv": hkv, "d": d, "causal": True, "dtype": dtype}
    samples = rng.choice([1, 1, 2, 5, 9])
    if form == "cross":
        nk = _log_int(rng, 64, 5_000)
        nq = _log_int(rng, 64, min(120_000, MOST // (nk * hq * d)))
    else:
        nq = nk = _log_int(rng, 32, min(50_000, int(math.sqrt(MOST / (hq * d)))))
    return {"op": op, "nq": nq, "nk": nk, "samples": samples, "hq": hq, "hkv": hkv, "d": d, "causal": form == "causal",
            "dtype": dtype}


def _lengths(n, samples):
    """n rows over the samples: one of a single row among three or more, an empty one among five or
    more, the others of unequal size."""
    fixed = {}
    if samples >= 3:
        fixed[1] = 1
    if samples >= 5:
        fixed[3] = 0
    rest = [i for i in range(samples) if i not in fixed]
    left = n - sum(fixed.values())
    weights = [3 + (5 * i) % 7 for i in range(len(rest))]
    sizes = [left * w // sum(weights) for w in weights]
    sizes[-1] += left - sum(sizes)
    out = [fixed.get(i, 0) for i in range(samples)]
    for i, s in zip(rest, sizes):
        out[i] = s
    return out


def _offsets(lengths):
    out = [0]
    for m in lengths:
        out.append(out[-1] + m)
    return out


def _bounds(case):
    """Row offsets of the samples in q and in k. Where every sample has the same few new tokens, only
    the caches are ragged."""
    if case["nq"] < case["nk"] and case["nq"] % case["samples"] == 0 and case["nq"] // case["samples"] <= 8:
        each = case["nq"] // case["samples"]
        return [each * i for i in range(case["samples"] + 1)], _offsets(_lengths(case["nk"], case["samples"]))
    return _offsets(_lengths(case["nq"], case["samples"])), _offsets(_lengths(case["nk"], case["samples"]))


def _pairs(case):
    return [case["d"] // 2 // case["axes"]] * case["axes"]


# ---- inputs -----------------------------------------------------------------------------------
def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    if case["op"] == "group_norm":
        n, c = case["n"], case["c"]
        x = randn(n, c)
        x.mul_(0.5 + torch.rand(c, generator=gen, device=dev)).add_(randn(c))
        bounds = _offsets(_lengths(n, case["samples"]))
        return {"x": x.to(DTYPES[case["dtype"]]), "gamma": 1 + 0.2 * randn(c), "beta": 0.2 * randn(c), "bounds": bounds,
                "offsets": torch.tensor(bounds, dtype=torch.int32, device=dev)}
    if case["op"] == "rope":
        n, hq, hk, d, dt = case["n"], case["hq"], case["hk"], case["d"], DTYPES[case["dtype"]]
        pos = torch.randint(0, case["grid"], (n, case["axes"]), generator=gen, device=dev, dtype=torch.int32)
        s = {"q": randn(n, hq, d).to(dt), "k": randn(n, hk, d).to(dt), "pos": pos, "q_gamma": None, "k_gamma": None}
        if case["norm"]:
            s["q_gamma"], s["k_gamma"] = 1 + 0.2 * randn(hq, d), 1 + 0.2 * randn(hk, d)
        return s
    hq, hkv, d, dt = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    qb, kb = _bounds(case)
    return {"q": randn(case["nq"], hq, d).to(dt), "k": randn(case["nk"], hkv, d).to(dt), "v": randn(case["nk"], hkv, d).to(dt),
            "q_bounds": qb, "k_bounds": kb, "q_offsets": torch.tensor(qb, dtype=torch.int32, device=dev),
            "k_offsets": torch.tensor(kb, dtype=torch.int32, device=dev)}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:     # what a program keeps from call to call: output buffers and workspaces
        pkg = _package()
        dev = torch.device("cuda")
        if case["op"] == "group_norm":
            state["result"] = torch.empty((case["n"], case["c"]), dtype=DTYPES[case["out"]], device=dev)
            state["workspace"] = pkg.group_norm_workspace(case["n"], case["c"], case["groups"], case["samples"], dev)
        elif case["op"] == "rope":
            state["q_result"], state["k_result"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
        else:
            state["result"] = torch.empty_like(state["q"])
            state["workspace"] = pkg.attention_workspace(case["nq"], case["nk"], case["samples"], case["hq"], case["hkv"],
                                                         case["d"], dev)
    return state


# ---- one pass ---------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        pkg = _package()
        if case["op"] == "group_norm":
            return pkg.group_norm(state["x"], case["groups"], state["gamma"], state["beta"], eps=EPS, silu=case["silu"],
                                  offsets=state["offsets"], out=state["result"], workspace=state["workspace"])
        if case["op"] == "rope":
            return pkg.rope_axes(state["q"], state["pos"], k=state["k"], pairs=_pairs(case), theta=THETA,
                                 interleaved=case["interleaved"], q_gamma=state["q_gamma"], k_gamma=state["k_gamma"], eps=EPS,
                                 q_out=state["q_result"], k_out=state["k_result"])
        return pkg.attention(state["q"], state["k"], state["v"], q_offsets=state["q_offsets"], k_offsets=state["k_offsets"],
                             causal=case["causal"], out=state["result"], workspace=state["workspace"])
    if case["op"] == "group_norm":
        return _plain_group_norm(state, case)
    if case["op"] == "rope":
        return _plain_rope(state, case)
    return _plain_attention(state, case)


def _plain_group_norm(state, case):
    g = case["groups"]
    parts = []
    for a, b in zip(state["bounds"], state["bounds"][1:]):
        if a == b:
            continue
        x = state["x"][a:b].float().reshape(b - a, g, -1)
        mean = x.mean(dim=(0, 2), keepdim=True)
        x = x - mean
        var = (x * x).mean(dim=(0, 2), keepdim=True)
        y = (x / torch.sqrt(var + EPS)).reshape(b - a, -1) * state["gamma"] + state["beta"]
        if case["silu"]:
            y = y / (1 + torch.exp(-y))
        parts.append(y.to(DTYPES[case["out"]]))
    return torch.cat(parts)


def _plain_rope(state, case):
    d = case["d"]
    angles = []
    for a, pairs in enumerate(_pairs(case)):
        exponent = -torch.arange(pairs, device=state["pos"].device, dtype=torch.float64) / pairs
        angles.append(state["pos"][:, a, None].double() * THETA ** exponent)
    angle = torch.cat(angles, dim=1)                   # in 64 bits: a far position's turn needs them
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turned = angle.shape[1]
    out = []
    for x, gamma in ((state["q"], state["q_gamma"]), (state["k"], state["k_gamma"])):
        y = x.float()
        if gamma is not None:
            y = y / torch.sqrt((y * y).mean(dim=-1, keepdim=True) + EPS) * gamma
        first, second = (y[..., 0::2], y[..., 1::2]) if case["interleaved"] else (y[..., : d // 2], y[..., d // 2:])
        u, w = first[..., :turned], second[..., :turned]
        first = torch.cat([u * cos - w * sin, first[..., turned:]], dim=-1)
        second = torch.cat([w * cos + u * sin, second[..., turned:]], dim=-1)
        y = torch.stack([first, second], dim=-1).flatten(-2) if case["interleaved"] else torch.cat([first, second], dim=-1)
        out.append(y.to(x.dtype))
    return out


def _plain_attention(state, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    share = hq // hkv
    out = torch.zeros_like(state["q"])
    for qa, qb, ka, kb in zip(state["q_bounds"], state["q_bounds"][1:], state["k_bounds"], state["k_bounds"][1:]):
        nq, nk = qb - qa, kb - ka
        if nq == 0 or nk == 0:
            continue
        k = state["k"][ka:kb].float().permute(1, 2, 0).contiguous()          # [hkv, d, nk]
        v = state["v"][ka:kb].float().permute(1, 0, 2).contiguous()          # [hkv, nk, d]
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
    qb, kb = _bounds(case)
    total = 0
    for qa, qe, ka, ke in zip(qb, qb[1:], kb, kb[1:]):
        nq, nk = qe - qa, ke - ka
        if not case["causal"]:
            total += nq * nk
        else:               # row i sees max(0, nk - nq + i + 1) keys
            first = max(0, nk - nq + 1)
            rows = min(nq, nk)
            total += rows * (first + nk) // 2 if rows else 0
    return total


def work(case):
    if case["op"] == "group_norm":
        e = case["n"] * case["c"]
        return {"bytes": e * (SIZE[case["dtype"]] + SIZE[case["out"]]) + 8 * case["c"], "flops": (12 if case["silu"] else 8) * e}
    if case["op"] == "rope":
        e = case["n"] * (case["hq"] + case["hk"]) * case["d"]
        gamma = 4 * (case["hq"] + case["hk"]) * case["d"] if case["norm"] else 0
        return {"bytes": 2 * e * SIZE[case["dtype"]] + 4 * case["n"] * case["axes"] + gamma, "flops": (7 if case["norm"] else 3) * e}
    rows = 2 * case["nq"] * case["hq"] + 2 * case["nk"] * case["hkv"]
    return {"bytes": rows * case["d"] * SIZE[case["dtype"]], "flops": 4 * case["d"] * case["hq"] * _visible(case)}


# ---- the definitions in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "group_norm":
        n, c, g = case["n"], case["c"], case["groups"]
        out = torch.empty((n, c), dtype=torch.float64, device=s["x"].device)
        for a, b in zip(s["bounds"], s["bounds"][1:]):
            for j in range(g):
                cols = slice(j * (c // g), (j + 1) * (c // g))
                x = s["x"][a:b, cols].double()
                if x.numel() == 0:
                    continue
                var, mean = torch.var_mean(x, unbiased=False)
                y = (x - mean) * torch.rsqrt(var + EPS) * s["gamma"][cols].double() + s["beta"][cols].double()
                out[a:b, cols] = y * torch.sigmoid(y) if case["silu"] else y
        return out
    if case["op"] == "rope":
        d = case["d"]
        turn = torch.ones((case["n"], d // 2), dtype=torch.complex128, device=s["pos"].device)
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
        return out
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.zeros((case["nq"], hq, d), dtype=torch.float64, device=s["q"].device)
    for qa, qe, ka, ke in zip(s["q_bounds"], s["q_bounds"][1:], s["k_bounds"], s["k_bounds"][1:]):
        if ke == ka:
            continue
        step = max(1, (1 << 27) // (ke - ka))
        for h in range(hq):
            k, v = s["k"][ka:ke, h * hkv // hq].double(), s["v"][ka:ke, h * hkv // hq].double()
            for a in range(qa, qe, step):
                b = min(qe, a + step)
                scores = s["q"][a:b, h].double() @ k.t() / math.sqrt(d)
                if case["causal"]:
                    i = torch.arange(a - qe, b - qe, device=scores.device)      # counted from the end
                    j = torch.arange(ka - ke, 0, device=scores.device)
                    scores = scores.masked_fill(j[None] > i[:, None], -math.inf)
                seen = torch.isfinite(scores).any(dim=1, keepdim=True)
                p = torch.softmax(torch.where(seen, scores, torch.zeros_like(scores)), dim=1)
                out[a:b, h] = torch.where(seen, p @ v, torch.zeros_like(out[a:b, h]))
    return out
