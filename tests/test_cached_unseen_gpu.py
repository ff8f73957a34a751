"""Values that are not finite reach every row that sees them, however small their weight, and no row that does not."""

from __future__ import annotations

import pytest
import torch

from plain_cached import E4M3, Case
from test_cached_attention_gpu import BF16, DEV, F32, check, queries, sets  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind, dtype, cache, dim, vdim", [
    ("tree", F32, F32, 48, 48), ("tree", F32, E4M3, 128, 128), ("single", F32, E4M3, 64, 64), ("single", BF16, E4M3, 32, 24),
    ("tree", BF16, BF16, 48, 40), ("tree", BF16, BF16, 128, 128), ("tree", BF16, E4M3, 64, 64), ("single", BF16, E4M3, 128, 128),
])
@pytest.mark.parametrize("value, below", [(float("nan"), 20.0), (float("nan"), 130.0), (float("nan"), 400.0), (float("inf"), 20.0)])
def test_values_that_are_not_finite_behind_small_weights(sets, kind, dtype, cache, dim, vdim, value, below):  # noqa: F811
    """A score 130 or 400 below the largest: a weight of 10^-57 or 10^-174, 0 in float32.  (Infinities stand before larger weights only: times
    such a one they are NaN in float32 and infinite in 64 bits.)"""
    if value == float("inf") and cache == E4M3:
        pytest.skip("a row of an 8-bit cache that held an infinity reads as NaN")
    case = Case(kind, [(200, 1), (40, 1)] if kind == "single" else [(200, [-1, 0, 0]), (40, [-1])], 1, dim, vdim, 16, cache, dtype, DEV, seed=7)
    q = queries(case, 2, dtype)
    q.fill_(1.0)
    case.kv.k.view(torch.uint8 if cache == E4M3 else dtype).zero_()  # (scores of 0 but for one)
    page, row = int(case.table[case.seats[0], 77 // 16]), 77 % 16
    if cache == E4M3:
        case.kv.k_scale.fill_(1.0)
        case.kv.k[page, 0, row] = -1.0
        case.kv.k_scale[page, 0, row] = below / dim**0.5
        case.kv.v_scale[page, 0, row] = value
    else:
        case.kv.k[page, 0, row] = -below / dim**0.5
        case.kv.v[page, 0, row, :3] = value
    if below == 400.0:  # (and a row that does not see the key, by its window)
        window = 60
        got = check(sets[dtype], case, 2, q, window=window)
        assert bool(torch.isfinite(got).all())
    got = check(sets[dtype], case, 2, q)
    first = torch.tensor([case.step.token_seq[t].item() == 0 for t in range(case.step.num_tokens)])
    assert bool((~torch.isfinite(got[first][:, :3])).all()) and bool(torch.isfinite(got[~first]).all())
