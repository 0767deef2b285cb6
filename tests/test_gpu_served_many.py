"""GPU test of as many samples as their count holds."""
from __future__ import annotations

import pytest

from test_gpu_served import gen, ints, same

pytestmark = pytest.mark.gpu


def test_rows_of_the_last_of_most_samples(gpu_lib):
    """Three rows of the last of 2^31 - 2 samples, and one between: appended and gathered as the samples of a call of two."""
    import torch
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GiB of device memory")
    samples, between = (1 << 31) - 2, 123_456_789
    offsets = torch.zeros(samples + 1, dtype=torch.int32, device="cuda")
    offsets[between + 1:] = 1
    offsets[-1] = 4
    lengths = torch.zeros(samples, dtype=torch.int32, device="cuda")
    lengths[between], lengths[-1] = 5, 10
    table = torch.full((samples, 1), -1, dtype=torch.int32, device="cuda")
    table[between], table[-1] = 1, 0
    k, v = gen(1)(4, 2, 64).bfloat16(), gen(2)(4, 2, 64).bfloat16()
    one, two = gpu_lib.kv_cache(2, 16, 2, 64), gpu_lib.kv_cache(2, 16, 2, 64)
    gpu_lib.kv_append(one, k, v, table, lengths, offsets=offsets)
    few = (ints([[1], [0]]), ints([5, 10]))
    gpu_lib.kv_append(two, k, v, *few, offsets=ints([0, 1, 4]))
    assert same(one.data, two.data) and bool((one.data != 0).any())
    a, b = gpu_lib.kv_gather(one, table, lengths, offsets=offsets, n=4), gpu_lib.kv_gather(two, *few, offsets=ints([0, 1, 4]), n=4)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
