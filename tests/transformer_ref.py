"""Plain 64-bit forms of the transformer pieces (group norm, rotary positions, attention) and the bounds
of what rounding may change, for the tests. Bounds count half steps of the output's type (torch.finfo(t).eps
/ 2) and the fp32 arithmetic before it."""
from __future__ import annotations

import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def offsets_of(lengths, start=0):
    out = [start]
    for m in lengths:
        out.append(out[-1] + m)
    return out


def group_norm(x, groups, bounds, gamma, beta, eps, silu):
    """-> (y, slack) in 64 bits, NaN outside the samples. slack is the fp32 arithmetic's part of the bound:
    2^-18 of the normalised value and of mean / std (sums of up to some hundred terms a thread, each
    rounded once: far below 2^6 of them in error at once; the mean is rounded to fp32), silu's slope is
    below 1.1."""
    n, c = x.shape
    y = torch.full((n, c), math.nan, dtype=torch.float64, device=x.device)
    slack = torch.zeros_like(y)
    g = torch.ones(c, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    for a, e in zip(bounds, bounds[1:]):
        if a == e:
            continue
        v = x[a:e].double().reshape(e - a, groups, c // groups)
        mean = v.mean(dim=(0, 2), keepdim=True)
        std = ((v - mean).square().mean(dim=(0, 2), keepdim=True) + eps).sqrt()
        z = ((v - mean) / std).reshape(e - a, c)
        t = z * g + b
        y[a:e] = t / (1 + torch.exp(-t)) if silu else t
        slack[a:e] = 1.1 * ((z.abs() + 1 + ((mean.abs() / std).expand(1, groups, c // groups).reshape(1, c))) * g.abs() * 2.0 ** -18
                            + (t.abs() + b.abs()) * 2.0 ** -21)
    return y, slack


def rope(x, pos, pairs, theta, interleaved, gamma, eps):
    """-> (y, slack): a pair's length times 2^-20 (the angle to 2^-22, sine and cosine, two products and a
    sum, the norm's few roundings)."""
    n, h, d = x.shape
    y = x.double()
    if gamma is not None:
        y = y / (y.square().mean(dim=-1, keepdim=True) + eps).sqrt() * gamma.double()
    u, v = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., : d // 2], y[..., d // 2:])
    angle = torch.zeros((n, d // 2), dtype=torch.float64, device=x.device)
    p = 0
    for a, cnt in enumerate(pairs):
        for j in range(cnt):
            angle[:, p] = pos[:, a].double() * theta ** (-j / cnt)
            p += 1
    cs, sn = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    uu, vv, length = u * cs - v * sn, v * cs + u * sn, torch.hypot(u, v)
    if interleaved:
        return torch.stack([uu, vv], -1).flatten(-2), torch.stack([length, length], -1).flatten(-2) * 2.0 ** -20
    return torch.cat([uu, vv], -1), torch.cat([length, length], -1) * 2.0 ** -20


def attention(q, k, v, q_bounds, k_bounds, causal, scale):
    """-> (o, slack), NaN outside the samples. slack: every probability is rounded to the 16-bit type (half a
    step of it, and 2^-25 of the largest below f16's normal range) and comes from a score with fp32 rounding
    (2^-12 together), so what the sum of p |v| / sum p allows. fp32 heads: probabilities are not rounded; a
    score of standard normal rows is off by at most d 2^-24 scale sum |q k| < 2^-14 for d <= 128, and a sum over
    lk keys, two an addition, by lk 2^-25. Keys that a row does not see are left out."""
    nq, hq, d = q.shape
    hkv = k.shape[1]
    o = torch.full((nq, hq, d), math.nan, dtype=torch.float64, device=q.device)
    slack = torch.zeros_like(o)
    longest = max([b - a for a, b in zip(k_bounds, k_bounds[1:])], default=0)
    part = 2.0 ** -14 + longest * 2.0 ** -25 if q.dtype == torch.float32 else half_step(q.dtype) + 2.0 ** -12
    for qa, qe, ka, ke in zip(q_bounds, q_bounds[1:], k_bounds, k_bounds[1:]):
        lq, lk = qe - qa, ke - ka
        if lq == 0:
            continue
        for h in range(hq):
            g = h // (hq // hkv)
            qs, ks, vs = q[qa:qe, h].double(), k[ka:ke, g].double(), v[ka:ke, g].double()
            if not causal or lk == 0:
                if lk == 0:
                    o[qa:qe, h] = 0
                    continue
                p = torch.softmax(qs @ ks.t() * scale, dim=1)
                o[qa:qe, h], slack[qa:qe, h] = p @ vs, part * (p @ vs.abs())
                slack[qa:qe, h] += 2.0 ** -24 * vs.abs().sum(0) if q.dtype == torch.float16 else 0.0
                continue
            finite = bool(torch.isfinite(ks).all() and torch.isfinite(vs).all())
            s = qs @ torch.nan_to_num(ks, 0, 0, 0).t() * scale if finite else None
            if finite:
                i = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
                s = s.masked_fill(torch.arange(lk, device=q.device)[None] > i, -math.inf)
                seen = (i >= 0)
                p = torch.softmax(torch.where(seen, s, torch.zeros_like(s)), dim=1) * seen
                o[qa:qe, h], slack[qa:qe, h] = p @ vs, part * (p @ vs.abs())
                slack[qa:qe, h] += 2.0 ** -24 * vs.abs().sum(0) if q.dtype == torch.float16 else 0.0
                continue
            for i in range(lq):     # row by row over the keys that it sees
                m = min(lk, max(0, lk - lq + i + 1))
                if m == 0:
                    o[qa + i, h] = 0
                    continue
                p = torch.softmax(ks[:m] @ qs[i] * scale, dim=0)
                o[qa + i, h], slack[qa + i, h] = p @ vs[:m], part * (p @ vs[:m].abs()) + (2.0 ** -24 * vs[:m].abs().sum(0) if q.dtype == torch.float16 else 0.0)
    return o, slack


def check(out, ref, slack, what=""):
    """out against ref: half a step of out's type at ref and slack; NaN where ref is NaN, the same
    infinities. Rows whose ref is NaN because no sample holds them are the caller's to compare."""
    half = half_step(out.dtype) if out.dtype != torch.float64 else 0.0
    tiny = 2.0 ** -25 if out.dtype == torch.float16 else 1e-38
    o = out.double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(o), torch.isnan(ref)), f"{what}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(o[inf], ref[inf]), f"{what}: infinities"
    d, tol = (o - ref).abs()[fin], (half * (ref.abs() + slack) + slack + tiny)[fin]
    worst = (d / tol).max().item() if d.numel() else 0.0
    print(f"  {what}: worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{what}: error {worst:.3f} times its bound"
