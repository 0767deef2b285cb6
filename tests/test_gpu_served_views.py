"""GPU tests of the served block's calls on views that interleave in one buffer: they share no value, and are taken."""
from __future__ import annotations

import pytest

from test_gpu_served import gen, ints, make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 200])
def test_attention_cached_between_q(gpu_lib, rows):
    """out's heads beside q's in each row, and between q's."""
    import torch
    cache, table = make_cache(gpu_lib, [rows + 50], 16, 2, 64, "mx4", 1)
    q = gen(rows)(rows, 4, 64).bfloat16()
    want = gpu_lib.attention_cached(q, cache, table, ints([rows + 50]))
    for q_at, o_at in ((slice(0, 4), slice(4, 8)), (slice(0, 8, 2), slice(1, 8, 2))):
        both = torch.full((rows, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        both[:, q_at] = q
        gpu_lib.attention_cached(both[:, q_at], cache, table, ints([rows + 50]), out=both[:, o_at])
        assert torch.equal(both[:, o_at], want) and torch.equal(both[:, q_at], q)


@pytest.mark.parametrize("held", ["mx4", "bf16"])
def test_gather_into_one_buffer(gpu_lib, held):
    """Keys and values beside each other in a row, head by head in turn, and one after the other."""
    import torch
    cache, table = make_cache(gpu_lib, [90], 16, 2, 64, held, 2)
    k, v = gpu_lib.kv_gather(cache, table, ints([90]), n=90)
    row = torch.zeros((90, 4, 64), dtype=torch.bfloat16, device="cuda")
    after = torch.zeros((180, 2, 64), dtype=torch.bfloat16, device="cuda")
    for ko, vo in ((row[:, :2], row[:, 2:]), (row[:, ::2], row[:, 1::2]), (after[:90], after[90:]), (after[::2], after[1::2])):
        gpu_lib.kv_gather(cache, table, ints([90]), k_out=ko, v_out=vo)
        assert torch.equal(ko, k) and torch.equal(vo, v)


@pytest.mark.parametrize("held", ["mx4", "bf16"])
@pytest.mark.parametrize("rows", [3, 700])
def test_append_out_of_one_buffer(gpu_lib, held, rows):
    """q, k, v and q_out beside each other in a row, or q_out's heads between q's."""
    import torch
    cache, table = make_cache(gpu_lib, [rows], 16, 2, 64, held, 3, fill=False)
    q, k, v = gen(1)(rows, 4, 64).bfloat16(), gen(2)(rows, 2, 64).bfloat16(), gen(3)(rows, 2, 64).bfloat16()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None].contiguous()
    want = gpu_lib.kv_append(cache, k, v, table, ints([rows]), q=q, pos=pos)
    pages = cache.data.clone()
    for q_at, o_at in ((slice(0, 4), slice(4, 8)), (slice(0, 8, 2), slice(1, 8, 2))):
        one = torch.full((rows, 12, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        one[:, q_at], one[:, 8:10], one[:, 10:] = q, k, v
        cache.data.zero_()
        gpu_lib.kv_append(cache, one[:, 8:10], one[:, 10:], table, ints([rows]), q=one[:, q_at], pos=pos, q_out=one[:, o_at])
        assert torch.equal(one[:, o_at], want) and torch.equal(one[:, q_at], q) and torch.equal(cache.data, pages)


@pytest.mark.parametrize("rows", [3, 700])
def test_attention_between_q(gpu_lib, rows):
    """The packed attention: q, k, v and out beside each other in a row, and out's heads between q's."""
    import torch
    q, k, v = gen(1)(rows, 4, 64).bfloat16(), gen(2)(rows, 2, 64).bfloat16(), gen(3)(rows, 2, 64).bfloat16()
    want = gpu_lib.attention(q, k, v, causal=True)
    for q_at, o_at in ((slice(0, 4), slice(4, 8)), (slice(0, 8, 2), slice(1, 8, 2))):
        one = torch.full((rows, 12, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        one[:, q_at], one[:, 8:10], one[:, 10:] = q, k, v
        gpu_lib.attention(one[:, q_at], one[:, 8:10], one[:, 10:], causal=True, out=one[:, o_at])
        assert torch.equal(one[:, o_at], want) and torch.equal(one[:, q_at], q)


@pytest.mark.parametrize("rows", [3, 700])
def test_rope_between_q(gpu_lib, rows):
    """Rotary positions: q, k and the outputs beside each other in a row, in place, and an output's heads between q's."""
    import torch
    q, k = gen(1)(rows, 4, 64).bfloat16(), gen(2)(rows, 2, 64).bfloat16()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None].contiguous()
    wq, wk = gpu_lib.rope_axes(q, pos, k=k)
    for q_at, o_at in ((slice(0, 4), slice(4, 8)), (slice(0, 8, 2), slice(1, 8, 2)), (slice(0, 4), slice(0, 4))):
        one = torch.full((rows, 12, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        one[:, q_at], one[:, 8:10] = q, k
        gpu_lib.rope_axes(one[:, q_at], pos, k=one[:, 8:10], q_out=one[:, o_at], k_out=one[:, 10:])
        assert torch.equal(one[:, o_at], wq) and torch.equal(one[:, 10:], wk) and torch.equal(one[:, 8:10], k)
