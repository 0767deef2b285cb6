"""Cases and closed forms for the cached attention's line of work: with q = 0 every key that a row sees weighs the same, and with
values that are 1 in one channel for 32 keys at a time and 0 elsewhere (exact in 4 and in 16 bits) each output is a count of
keys over their number, so that one tile lost or counted twice moves its channel by more than any rounding."""
from __future__ import annotations

import torch

KEYS = 32       # in a row with one channel

# new rows, keys, hq, hkv, d, page, columns of the table (0: as many as it takes). Units of 16, 32 (4 bits alone) and 128 rows; joins by
# a group of lanes, a wave and a workgroup; weights in 64ths of a tile, in tiles and, with wide tables, in several tiles.
CASES = [
    ([1], [40_009], 8, 2, 128, 64, 0), ([1], [300_001], 8, 2, 128, 64, 0), ([1], [1_025], 4, 4, 128, 16, 0),
    ([1] * 5, [20_000, 0, 33, 150_001, 1], 8, 2, 128, 32, 0), ([1] * 40, [(i * 977) % 9000 + 1 for i in range(40)], 8, 2, 128, 64, 0),
    ([1] * 200, [(i * 677) % 1500 for i in range(200)], 4, 2, 128, 64, 0), ([1] * 64, [512] * 64, 16, 8, 64, 64, 0),
    ([3, 1, 2] * 5, [9001, 5, 20_033] * 5, 8, 2, 64, 16, 0), ([8], [40_009], 4, 1, 128, 128, 0), ([6], [20_033], 5, 1, 40, 32, 0),
    ([20] * 30, [3001] * 30, 2, 2, 96, 64, 0), ([20] * 30, [701 + 3 * i for i in range(30)], 8, 8, 96, 64, 0), ([30], [100_003], 1, 1, 128, 64, 0),
    ([2, 300, 1], [70_001, 40_009, 3], 8, 2, 128, 64, 0), ([40, 33], [300_007, 90_001], 4, 1, 128, 64, 0), ([70], [9001], 4, 4, 32, 16, 0),
    ([8001], [8001], 4, 1, 128, 64, 0), ([8001], [8001], 2, 1, 64, 64, 0), ([3000, 2001], [20_033, 3000], 4, 2, 128, 64, 0),
    ([2000, 1, 1, 900, 0, 1], [1030, 40_009, 0, 2000, 50, 7], 4, 2, 96, 32, 0), ([3000], [1029], 4, 4, 64, 64, 0), ([129], [400_009], 1, 1, 128, 256, 0),
    ([1] * 16, [7 + 999 * i for i in range(16)], 8, 2, 128, 256, 1 << 22), ([5], [70_001], 8, 2, 128, 256, 1 << 22),
    ([700, 900], [40_009, 900], 4, 4, 128, 256, 1 << 22),
]


def shift(s, head):
    """Where a sample's and key head's channels begin."""
    return 5 * s + 11 * head


def values(lengths, hkv, d):
    """[sum of lengths, hkv, d], packed."""
    j = torch.cat([torch.arange(n) // KEYS + shift(s, 0) for s, n in enumerate(lengths)] or [torch.zeros(0, dtype=torch.long)])
    channel = (j[:, None] + torch.tensor([shift(0, h) for h in range(hkv)])) % d
    return channel[..., None] == torch.arange(d)


def expected(limits, s, head, d, without=None, twice=None):
    """[rows, d] in 64 bits for rows that see so many keys (zeros where none); without, twice: a run of KEYS keys that is left out, or
    counted twice."""
    n = limits.double()[:, None]
    e = (torch.arange(d, device=limits.device) - shift(s, head)) % d        # the channel's place in a cycle
    full, rest = limits[:, None] // (KEYS * d), limits[:, None] % (KEYS * d)
    count = (full * KEYS + (rest - e * KEYS).clamp(0, KEYS)).double()
    for run, sign in ((without, -1), (twice, 1)):
        if run is not None:
            part = sign * (limits[:, None] - run * KEYS).clamp(0, KEYS).double()
            count, n = count + part * (e == run % d), n + part
    return torch.where(n > 0, count / n.clamp(min=1), torch.zeros_like(count))


def limits_of(m, n, causal):
    """What the rows of a sample with m rows and n keys see."""
    i = torch.arange(m)
    return (i + n - m + 1).clamp(0, n) if causal else torch.full_like(i, n)
