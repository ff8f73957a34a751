"""Attention over the cache for heads of every size the layers take: none is refused for the shared memory it asks for."""

from __future__ import annotations

import pytest

from plain_cached import E4M3, Case
from test_cached_attention_gpu import BF16, DEV, F32, check, sets  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

# Around 48 KB (heads of 140 to 156, or smaller keys with larger values and the other way round), and the ends of the range.
SIZES = [(d, d) for d in (1, 2, 112, 136, 140, 143, 144, 145, 148, 150, 151, 152, 153, 156, 160, 200, 255, 256)]
SIZES += [(80, 256), (76, 256), (84, 250), (256, 1), (1, 256), (256, 8), (200, 77), (180, 100), (100, 233), (136, 160)]


@pytest.mark.parametrize("dim, vdim", SIZES)
def test_heads_of_every_size(sets, dim, vdim):  # noqa: F811
    for dtype, cache in ((F32, F32), (F32, E4M3), (BF16, BF16), (BF16, E4M3)):
        check(sets[dtype], Case("tree", [(40, [-1, 0, 0, 1]), (3, [-1])], 2, dim, vdim, 16, cache, dtype, DEV, seed=dim), 4)
        if cache == E4M3:
            check(sets[dtype], Case("single", [(70, 1), (0, 1)], 2, dim, vdim, 16, cache, dtype, DEV, seed=vdim), 4)
