"""GPU tests of the cached attention where its line of work is cut and joined: no tile is lost or counted twice, whatever the
kernel, the join and the lengths."""
from __future__ import annotations

import pytest

import line_cases as lc
import transformer_ref as ref
from test_gpu_served import dtype, gen, ints

pytestmark = pytest.mark.gpu


def filled(pkg, case, held, key):
    """A cache with the case's values, its table (pages dealt at random)."""
    import torch
    new, lengths, hq, hkv, d, page, columns = case
    counts = [-(-n // page) for n in lengths]
    pool = sum(counts) + 1
    cache = pkg.kv_cache(pool, page, hkv, d, "mx4" if held == "mx4" else dtype(held))
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(page)).to(torch.int32)
    narrow = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32)
    at = 0
    for s, m in enumerate(counts):
        narrow[s, :m] = order[at: at + m]
        at += m
    table = torch.full((len(lengths), max(columns, max(counts))), -1, dtype=torch.int32, device="cuda")
    table[:, : max(counts)] = narrow.cuda()
    v = lc.values(lengths, hkv, d).to("cuda").to(dtype(key))
    k = gen(1)(*v.shape).to(dtype(key))
    pkg.kv_append(cache, k, v, table, ints(lengths), offsets=ints(ref.offsets_of(lengths)))
    return cache, table


@pytest.mark.parametrize("case", range(len(lc.CASES)))
@pytest.mark.parametrize("held,key", [("mx4", "bf16"), ("mx4", "f16"), ("bf16", "bf16")])
def test_no_tile_is_lost(gpu_lib, case, held, key):
    """A row's sums are whole numbers of equal weights, which fp32 holds: the division (2^-22) and the output's rounding are all that
    may be off."""
    import torch
    new, lengths, hq, hkv, d, page, columns = lc.CASES[case]
    print(f"[line] {case} held {held} {key}", flush=True)
    cache, table = filled(gpu_lib, lc.CASES[case], held, key)
    b = ref.offsets_of(new)
    q = torch.zeros((sum(new), hq, d), dtype=dtype(key), device="cuda")
    for causal in (True, False):
        out = gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints(b), causal=causal)
        want = torch.empty((sum(new), hq, d), dtype=torch.float64, device="cuda")
        for s, (m, n) in enumerate(zip(new, lengths)):
            for h in range(hq if m else 0):
                want[b[s]: b[s + 1], h] = lc.expected(lc.limits_of(m, n, causal).cuda(), s, h * hkv // hq, d)
        ref.check(out, want, want * 2.0 ** -21, f"causal={causal}")
