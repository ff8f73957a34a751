"""Numbers next to a border of e4m3: every kernel that stores them rounds alike."""

from __future__ import annotations

import pytest
import torch

from plain_cached import E4M3, MOST, Case
from test_cached_attention_gpu import BF16, DEV, F32, sets  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def near_borders(n, seed):
    """(rows of n numbers, the e4m3 numbers that each over its row's scale is nearest to, in float32 arithmetic): numbers next to a
    border, for which multiplying by the scale's reciprocal and dividing by the scale give different ones."""
    g = torch.Generator().manual_seed(seed)
    most = torch.exp2(torch.rand(400, 1, generator=g) * 12 - 6)
    scale = most / MOST
    numbers = torch.arange(2, 126, dtype=torch.uint8).view(E4M3).float()
    borders = (numbers[:-1] + numbers[1:]) / 2
    x = (borders * scale).repeat(1, 9)
    x = (x.view(torch.int32) + torch.arange(-4, 5, dtype=torch.int32).repeat_interleave(borders.numel())).view(torch.float32)
    apart = (x / scale).to(E4M3).view(torch.uint8) != (x * (1 / scale)).to(E4M3).view(torch.uint8)
    rows = []
    for r in range(most.shape[0]):
        found = x[r][apart[r] & (x[r] < most[r])]
        if found.numel() >= 4:
            row = torch.zeros(n)
            row[0] = most[r]
            row[1 : 1 + min(n - 1, found.numel())] = found[: n - 1]
            rows.append(row)
    rows = torch.stack(rows)
    return rows, (rows / (rows.amax(-1, keepdim=True) / MOST)).to(E4M3)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [128, 64, 48])
def test_numbers_next_to_a_border_are_divided(sets, dtype, dim):  # noqa: F811
    """A number is the row's over its scale, whichever kernel stores it."""
    rows, want = near_borders(dim, 3)
    tokens = rows.shape[0]
    assert tokens > 50
    case = Case("portion", [(11, tokens)], 1, dim, dim, 16, E4M3, dtype, DEV)
    rows = rows.to(DEV)
    sets[dtype].kv_write(rows, rows, case.step, case.kv)
    sets[dtype].check_errors()
    places = range(11, 11 + tokens)
    table = case.table[case.seats[0]]
    for held in (case.kv.k, case.kv.v):
        got = torch.stack([held.view(torch.uint8)[int(table[p // 16]), 0, p % 16] for p in places]).cpu()
        assert torch.equal(got, want.view(torch.uint8))
