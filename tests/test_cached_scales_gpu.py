"""Rows of 8-bit caches whose scales are as far apart as they can be."""

from __future__ import annotations

import pytest
import torch

from plain_cached import E4M3, MOST, Case
from test_cached_attention_gpu import BF16, DEV, check, queries, sets  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim, heads", [(128, 6), (64, 12), (48, 4)])
@pytest.mark.parametrize("large", [2.0**40, 2.0**115])
def test_a_key_without_weight_whose_value_is_huge(sets, dim, heads, large):  # noqa: F811
    """Values of 2^-100 and, behind a score of minus some thousands or a mask, others that are up to 2^215 times as large: they have no weight."""
    k = sets[BF16]
    case = Case("single", [(300, 1), (40, 1)], 2, dim, dim, 16, E4M3, BF16, DEV, seed=1)
    q = queries(case, heads, BF16)
    q.abs_().add_(0.5)
    case.kv.v_scale.fill_(2.0**-100)
    for request, key in ((0, 200), (0, 290), (1, 33)):
        page = int(case.table[case.seats[request], key // 16])
        case.kv.k[page, :, key % 16] = -MOST  # (q is positive: below every other score by thousands)
        case.kv.k_scale[page, :, key % 16] = 8.0
        case.kv.v_scale[page, :, key % 16] = large
    got = check(k, case, heads, q)
    assert bool(torch.isfinite(got).all()) and float(got.abs().max()) < 2.0**-80
    # A tree whose second branch holds such a value: the first does not see it.
    case = Case("tree", [(300, [-1, 0, -1, 1]), (2, [-1, -1])], 2, dim, dim, 16, E4M3, BF16, DEV, seed=2)
    case.kv.v_scale.fill_(2.0**-100)
    for request, place in ((0, 302), (1, 3)):
        case.kv.v_scale[int(case.table[case.seats[request], place // 16]), :, place % 16] = large
    got = check(k, case, heads)
    apart = torch.tensor([t not in (2, 5) for t in range(6)])  # (tokens 2 and 5 see their own)
    assert bool(torch.isfinite(got).all()) and float(got[apart].abs().max()) < 2.0**-80 and float(got[~apart].abs().min()) > 0.0
