"""GPU tests of the 8-bit linear on products that every form of its sum holds exactly, where one lost product shows; and of
the cached attention's scale."""
from __future__ import annotations

import pytest

import served_ref as sr
import transformer_ref as ref
from test_gpu_served import ATTEND_CASES, LINEAR_CASES, dtype, gen, ints, make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,ci,co", LINEAR_CASES)
@pytest.mark.parametrize("ok", ["bf16", "f16", "f32"])
def test_linear_mx_of_ones(gpu_lib, n, ci, co, ok):
    """x and W of 0, 1 and -1, a block's power in the one its inverse in the other: every product is 0, 1 or -1, every sum of up to
    4,096 of them a whole number that is within 16 bits of one product, whichever instruction adds. The output is that number,
    rounded once (whole numbers up to 256 are bf16's, up to 2,048 fp16's)."""
    import torch
    print(f"[linear of ones] {n} x {ci} -> {co} {ok}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(n + ci + co)
    x, w = (torch.randint(0, 2, (m, ci), generator=g, device="cuda") * (2 * torch.randint(0, 2, (m, ci), generator=g, device="cuda") - 1)
            for m in (n, co))
    x, w = x.float(), w.float()
    scale = torch.exp2(torch.randint(-6, 7, (ci // 32,), generator=g, device="cuda").float()).repeat_interleave(32)
    out = gpu_lib.linear_mx(gpu_lib.Mx(*sr.to_mx(x * scale)), gpu_lib.Mx(*sr.to_mx(w / scale)), out_dtype=dtype(ok))
    want = x.double() @ w.double().t()
    assert torch.equal(out, want.to(dtype(ok))), int((out != want.to(dtype(ok))).sum())


@pytest.mark.parametrize("scale", [0.01, 1.0])
@pytest.mark.parametrize("case", [4, 6, 7, 10, 13, 14])
@pytest.mark.parametrize("held,key", [("mx4", "bf16"), ("mx4", "f16"), ("bf16", "bf16")])
def test_attention_cached_scale(gpu_lib, case, scale, held, key):
    new, lengths, hq, hkv, d, page = ATTEND_CASES[case]
    print(f"[scale] {case} {scale} held {held} {key}", flush=True)
    cache, table = make_cache(gpu_lib, lengths, page, hkv, d, held, case)
    q = gen(case)(sum(new), hq, d).to(dtype(key))
    b = ref.offsets_of(new)
    out = gpu_lib.attention_cached(q, cache, table, ints(lengths), offsets=ints(b), scale=scale)
    o, slack = sr.attention_cached(q, cache, table, lengths, b, True, scale)
    ref.check(out, o, slack, "attention")
