"""Tokens of a step of drafted tokens that belong to no request: their rows of the output are left as they were."""

from __future__ import annotations

from dataclasses import replace

import pytest
import torch

from plain_cached import E4M3, Case, half_step, random_parents
from test_cached_attention_gpu import BF16, DEV, F32, queries, sets  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

FEW = [(5000, random_parents(9, 1)), (40, random_parents(7, 2)), (900, [-1, 0])]   # keys in several shares
MANY = [(130, random_parents(5, i)) for i in range(40)]                             # one share


def poisoned_memory():
    held = [torch.full((1 << 24,), float("nan"), device=DEV), *(torch.full((1 << 17,), float("nan"), device=DEV) for _ in range(8))]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("dtype, cache, dim, heads", [(BF16, BF16, 128, 12), (BF16, E4M3, 64, 6), (BF16, BF16, 48, 4), (F32, F32, 64, 4), (F32, E4M3, 32, 8)])
@pytest.mark.parametrize("requests", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("what", ["shorter", "empty", "most", "all"])
def test_tokens_of_no_request(sets, dtype, cache, dim, heads, requests, what):  # noqa: F811
    k = sets[dtype]
    case = Case("tree", requests, 2, dim, dim, 16, cache, dtype, DEV, seed=3)
    q, tree = queries(case, heads, dtype), case.step.tree
    seqs, most, lengths = tree.seqs.clone(), tree.most_nodes, list(case.news)
    if what == "shorter":  # a padded request: its last tokens are nobody's
        lengths[0] -= 2
    elif what == "empty":
        lengths[-1] = 0
    elif what == "most":  # more of a request's tokens than the step says there are at most
        most, lengths = 3, [min(n, 3) for n in lengths]
    else:
        lengths = [0] * len(lengths)
    if what != "most":
        seqs[:, 1] = torch.tensor(lengths, dtype=torch.int32)
    step = replace(case.step, tree=replace(tree, seqs=seqs, most_nodes=most))
    out = torch.full((step.num_tokens, heads * dim), 7.0, dtype=dtype, device=DEV)
    poisoned_memory()
    k.attention(q, out, step, case.kv, heads, 2, dim, None, dim**-0.5)
    k.check_errors()
    kept = torch.tensor([j < lengths[r] for r, n in enumerate(case.news) for j in range(n)])
    got = out.double().cpu()
    assert bool((got[~kept] == 7.0).all())
    want, size = case.attention(q, heads, dim**-0.5)
    # (as in the tests of whole steps: the output's rounding, the weights' to 16 bits, float32 sums and exponentials)
    slack = half_step(dtype) * want.abs() + ((half_step(BF16) if dtype == BF16 else 0.0) + 2.0**-15) * size
    slack = slack + (case.least if dtype == BF16 else 0.0)
    assert bool(((got - want).abs() <= slack)[kept].all())
