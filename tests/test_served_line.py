"""CPU tests of the closed forms that the cached attention's line is tested with: they are what counting gives, and a run of keys
that is lost or counted twice is past the bound."""
from __future__ import annotations

import pytest
import torch

import line_cases as lc


def test_expected_is_a_count():
    for n, d, s, head in ((1, 8, 0, 0), (33, 8, 2, 1), (700, 16, 1, 3), (5000, 40, 7, 0), (4096, 32, 0, 5)):
        v = lc.values([0] * s + [n], head + 1, d)[:, head].double()
        limits = torch.tensor([0, 1, 31, 32, 33, n // 2, n]).clamp(max=n)
        want = torch.stack([v[:m].mean(0) if m else torch.zeros(d, dtype=torch.float64) for m in limits.tolist()])
        assert torch.allclose(lc.expected(limits, s, head, d), want, rtol=1e-12, atol=0)


@pytest.mark.parametrize("case", range(len(lc.CASES)))
def test_a_lost_run_shows(case):
    """With the kernel's answer as near to the wrong value as rounding may bring it to the right one, in bf16."""
    new, lengths, hq, hkv, d, page, columns = lc.CASES[case]
    for s, (m, n) in enumerate(zip(new, lengths)):
        if m == 0 or n < 2 * lc.KEYS:
            continue
        limits = lc.limits_of(m, n, True)[-1:]
        want = lc.expected(limits, s, 0, d)
        for run in (0, n // lc.KEYS // 2, n // lc.KEYS - 1):
            for wrong in (lc.expected(limits, s, 0, d, without=run), lc.expected(limits, s, 0, d, twice=run)):
                assert bool(((wrong - want).abs() > 2.0 ** -8 * (wrong + want) + 2.0 ** -20 * want).any()), (case, s, run)
