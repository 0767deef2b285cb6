"""Plain 64-bit forms of a served block's pieces (RMS norm, numbers of few bits, the paged cache, attention to it) and the
bounds of what rounding may change, for the tests."""
from __future__ import annotations

import math

import torch

import transformer_ref as ref

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---- numbers of few bits ------------------------------------------------------------------------
def power_of(amax, most):
    """The power byte of blocks with that largest value (float64): the least 2^e with amax <= most 2^e; 255 where it is
    not finite."""
    fin = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(fin, amax, torch.ones_like(amax)) / most)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    return torch.where(fin, (e + 127).clamp(min=0), torch.full_like(e, 255)).to(torch.uint8)


def scale_of(power):
    """2^(power - 127) in 64 bits, NaN for 255."""
    p = power.to(torch.float64)
    return torch.where(power == 255, torch.full_like(p, math.nan), torch.exp2(p - 127))


def blocked(x):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))


def amax_of(x):
    a = blocked(x.double()).abs()
    bad = ~torch.isfinite(a)
    return torch.where(bad.any(-1), torch.full_like(a[..., 0], math.inf), torch.where(bad, torch.zeros_like(a), a).amax(-1))


def round_e4m3(y):
    """Float64 values of at most 448 to the nearest e4m3 value, halfway to the even code."""
    a = y.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(a / step) * step, y)


def round_e2m1(y):
    a = y.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=1.0))) - 1)
    return torch.copysign(torch.round(a / step) * step, y)


def of_mx(mx):
    """An Mx's values in 64 bits."""
    codes, powers = mx
    return (blocked(codes.double()) * scale_of(powers.view(torch.uint8))[..., None]).flatten(-2)[..., : codes.shape[1]]


def to_mx(x):
    """Any values as an Mx (float8_e4m3fn, float8_e8m0fnu) by these rules."""
    power = power_of(amax_of(x), 448.0)
    y = torch.nan_to_num((blocked(x.double()) / scale_of(power)[..., None]).flatten(-2), 0, 0, 0)
    return round_e4m3(y).to(torch.float32).to(torch.float8_e4m3fn), power.view(torch.float8_e8m0fnu)


def mx4_values(x):
    """x [..., d] as its 4-bit codes stand for it, in 64 bits."""
    b = blocked(x.double())
    s = scale_of(power_of(amax_of(x), 6.0))[..., None]
    return (round_e2m1(b / s) * s).flatten(-2)[..., : x.shape[-1]]


# ---- norm and linear -----------------------------------------------------------------------------
def rms_norm(x, residual, gamma, eps):
    """-> (y, h) in 64 bits. The fp32 arithmetic's part of the bound is 2^-18 of y: a sum of up to 2^5 squares a lane
    and 2^5 more additions, half of whose error the root keeps, and six roundings."""
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / (h.square().mean(dim=1, keepdim=True) + eps).sqrt()
    return (y if gamma is None else y * gamma.double()), h


NORM_SLACK = 2.0 ** -18


def linear(x, w, bias, act, residual, exact):
    """x and w values in 64 bits -> (y, slack). fp32 sums of ci products: at most ci 2^-24 of the products' sizes' sum. The 8-bit
    matrix instruction keeps some 16 bits below the largest of its products: 2^-12 of that sum."""
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    slack = size * (x.shape[1] * 2.0 ** -24 if exact else 2.0 ** -12)
    if bias is not None:
        z = z + bias.double()
        slack = slack + 2.0 ** -23 * (z.abs() + bias.double().abs())
    if act == "silu":
        z = torch.where(z == -math.inf, torch.full_like(z, math.nan), z * torch.sigmoid(z))
        slack = 1.1 * slack + 2.0 ** -20 * z.abs()
    if residual is not None:
        z = z + residual.double()
        slack = slack + 2.0 ** -23 * (z.abs() + residual.double().abs())
    return z, slack


# ---- the cache -----------------------------------------------------------------------------------
def decode(cache):
    """K and V [pages, page, heads, d] in 64 bits from a KVCache's bytes."""
    data, h, p, d = cache.data, cache.heads, cache.page, cache.d
    b = -(-d // 32)
    heads = data.reshape(data.shape[0], h, -1)
    out = []
    for side in range(2):
        if cache.dtype == "mx4":
            codes = heads[:, :, side * 16 * b * p: (side + 1) * 16 * b * p].reshape(-1, h, p, 16 * b).long()
            power = heads[:, :, (32 + side) * b * p: (33 + side) * b * p].reshape(-1, h, p, b)
            table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=data.device)
            x = torch.stack([table[codes & 15], table[codes >> 4]], -1).flatten(-2)
            x = (x.unflatten(-1, (b, 32)) * scale_of(power)[..., None]).flatten(-2)[..., :d]
        else:
            x = heads[:, :, side * 2 * d * p: (side + 1) * 2 * d * p].contiguous().view(cache.dtype).reshape(-1, h, p, d).double()
        out.append(x.transpose(1, 2))
    return out


def place(cache, table, s, j):
    """(page, slot) of key j of sample s, or None where the cache does not hold it."""
    if not 0 <= j < table.shape[1] * cache.page:
        return None
    page = int(table[s, j // cache.page])
    return (page, j % cache.page) if 0 <= page < cache.pages else None


def keys_of(cache, table, lengths, s):
    """(K, V [keys, heads, d] in 64 bits, held [keys]) of sample s; keys that the cache does not hold are zeros."""
    k, v = decode(cache)
    n = min(max(int(lengths[s]), 0), table.shape[1] * cache.page)
    if n == 0:
        z = torch.zeros((0, cache.heads, cache.d), dtype=torch.float64, device=k.device)
        return z, z, torch.zeros(0, dtype=torch.bool, device=k.device)
    j = torch.arange(n, device=k.device)
    page = table[s].to(k.device)[j // cache.page].long()
    held = (page >= 0) & (page < cache.pages)
    page = torch.where(held, page, torch.zeros_like(page))
    kk, vv = k[page, j % cache.page], v[page, j % cache.page]
    zero = torch.zeros((), dtype=torch.float64, device=k.device)
    return torch.where(held[:, None, None], kk, zero), torch.where(held[:, None, None], vv, zero), held


def attention_cached(q, cache, table, lengths, bounds, causal, scale):
    """-> (o, slack), NaN for rows outside the samples; slack as transformer_ref.attention's, over the keys that a row
    sees."""
    nq, hq, d = q.shape
    o = torch.full((nq, hq, d), math.nan, dtype=torch.float64, device=q.device)
    slack = torch.zeros_like(o)
    part = ref.half_step(q.dtype) + 2.0 ** -12
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 0.0
    for s, (a, e) in enumerate(zip(bounds, bounds[1:])):
        a, e = max(a, 0), min(e, nq)
        m = e - a
        if m <= 0:
            continue
        k, v, held = keys_of(cache, table, lengths, s)
        lk = k.shape[0]
        if lk == 0:
            o[a:e] = 0
            continue
        i, j = torch.arange(m, device=q.device)[:, None], torch.arange(lk, device=q.device)[None]
        sees = held[None] & ((j <= i + lk - m) if causal else torch.ones_like(j <= i))
        some = sees.any(1, keepdim=True)
        for h in range(hq):
            g = h * cache.heads // hq
            t = torch.where(sees, q[a:e, h].double() @ torch.nan_to_num(k[:, g], math.nan, math.inf, -math.inf).t() * scale
                            if bool(torch.isfinite(k[:, g]).all()) else (q[a:e, h].double()[:, None] * k[None, :, g]).sum(-1) * scale,
                            torch.full_like(sees, -math.inf, dtype=torch.float64))
            p = torch.softmax(torch.where(some, t, torch.zeros_like(t)), dim=1)
            p = torch.where(sees, p, torch.zeros_like(p))
            fin = torch.isfinite(v[:, g])
            vf = torch.where(fin, v[:, g], torch.zeros_like(v[:, g]))
            y = p @ vf
            for x in (~fin).any(1).nonzero().flatten().tolist():
                y += torch.where(sees[:, x, None] & ~fin[None, x], p[:, x, None] * v[x, g][None], torch.zeros_like(y))
            o[a:e, h] = y
            slack[a:e, h] = part * (p @ vf.abs()) + tiny * (sees.double() @ vf.abs())
    return o, slack
