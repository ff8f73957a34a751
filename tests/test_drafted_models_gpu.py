"""Drafted trees through models whose attention has windows, kept first keys, values that are the keys or of another size, sinks
and caps: the logits of every path, and whole generations, are those of ordinary steps."""

from __future__ import annotations

import pytest
import torch

import helpers
import test_fovudra as fovudra
import test_zuzunex as zuzunex
from plain_cached import random_parents
from test_cached_engine import path_to

from distie_b200.engine.batch import BatchEntry
from distie_b200.kernels import make_kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

_A, _MOE = fovudra._attention, fovudra._moe
FOVUDRA = {
    "architecture": "Fovudra", "vocab": 131, "width": 64, "norm": {"eps": 1e-5},
    "layers": [_A(4, 2, 16, 8, 1, 16, 1e4, None, 0.25, _MOE(3, 1, 20, None)), _A(6, 3, 64, 30, 9, 32, 1e6, None, 0.125, None),
               _A(2, 1, 128, 300, 2, 64, 100.0, None, 0.09, _MOE(2, 2, 24, 56)), _A(4, 4, 24, 7, 0, 24, 500.0, None, 0.2, None)],
}
_L = zuzunex._layer
ZUZUNEX = {
    "architecture": "Zuzunex", "vocab": 131, "width": 64, "norm": {"eps": 1e-5}, "loop": {"start": 0, "stop": 2, "times": 2},
    "layers": [_L("attention", zuzunex._plain(3, 3, 8, 10, 0.5, 5.0, (0.7, 5)), zuzunex._dense(40)),
               _L("attention_2", zuzunex._conv(4, 1, 128, 128, 0.09, None, (10000.0, 64), (4.0, 64, 8.0, 1.0)), None),
               _L("attention", zuzunex._plain(16, 1, 64, 64, 0.13, 20.0, None), None),
               _L("attention_2", zuzunex._conv(6, 3, 80, 48, 0.11, None, (10000.0, 80)), zuzunex._moe(4, 0, 2, 32, None))],
}


def engine_of(which, dtype, blocks=400, page=8, **knobs):
    tests, cfg = (fovudra, FOVUDRA) if which == "fovudra" else (zuzunex, ZUZUNEX)
    weights = (fovudra.pf if which == "fovudra" else zuzunex.pz).random_weights(cfg, 3)
    return tests.engine_of(cfg, weights, page, make_kernels(dtype, DEV), blocks, **knobs)


@pytest.mark.parametrize("which", ["fovudra", "zuzunex"])
@pytest.mark.parametrize("cache_dtype", ["auto", "float8_e4m3"])
def test_every_path_of_a_tree(which, cache_dtype):
    """The float32 engine: trees of two requests and a single token beside them, against the paths one after another."""
    engine = engine_of(which, torch.float32, max_seqs=8, cache_dtype=cache_dtype)
    prompts = [helpers.random_ids(131, n, 60 + n) for n in (45, 3, 20)]
    trees = [random_parents(30, 1), random_parents(11, 2), [-1]]
    drafts = [helpers.random_ids(131, len(t), 90 + i) for i, t in enumerate(trees)]
    seats = [engine.cache.open_seat() for _ in prompts]
    for seat, ids in zip(seats, prompts):
        assert engine.cache.grow(seat, len(ids) + 40)
        engine.runner.step([BatchEntry(seat, ids, 0, ())])
        engine.cache.trim(seat, len(ids))
    entries = [BatchEntry(s, d, len(p), tuple(range(len(d))), t) for s, d, p, t in zip(seats, drafts, prompts, trees)]
    entries[2].parents = None
    logits = engine.runner.step(entries).float().cpu()
    engine.runner.finish_step()
    at, worst = 0, 0.0
    for ids, draft, tree in zip(prompts, drafts, trees):
        leaves = [n for n in range(len(tree)) if n not in tree]
        for leaf in leaves:
            path = path_to(leaf, tree)
            seat = engine.cache.open_seat()
            assert engine.cache.grow(seat, len(ids) + len(path))
            engine.runner.step([BatchEntry(seat, ids, 0, ())])
            want = torch.cat([engine.runner.step([BatchEntry(seat, [draft[n]], len(ids) + i, (0,))]).float().cpu().clone() for i, n in enumerate(path)])
            engine.cache.close_seat(seat)
            got = logits[[at + n for n in path]]
            worst = max(worst, float((got - want).abs().max() / want.abs().max()))
        at += len(tree)
    # Sums in another order; over an 8-bit cache a number next to a border may go the other way (test_cached_engine says how far).
    assert worst <= (helpers.FP32_TOL if cache_dtype == "auto" else 0.05), worst


@pytest.mark.parametrize("which", ["fovudra", "zuzunex"])
@pytest.mark.parametrize("dtype, cache_dtype", [(torch.float32, "auto"), (torch.float32, "float8_e4m3"), (torch.bfloat16, "auto"), (torch.bfloat16, "float8_e4m3")])
def test_generations(which, dtype, cache_dtype):
    """Drafted generation in a pool that holds little more than the request, windows giving pages back on the way."""
    engine = engine_of(which, dtype, blocks=14, max_seqs=2, cache_dtype=cache_dtype, token_budget=32)
    prompt = helpers.random_ids(131, 40, 8)
    answer = engine.generate([prompt], max_new_tokens=40, ignore_eos=True)[0].token_ids

    def drafter(ids):
        at = len(ids) - len(prompt)
        right = answer[at : at + 6]
        wrong = [(t + 1) % 131 for t in right]
        return [t for pair in zip(wrong, right) for t in pair], [p for i in range(len(right)) for p in ((-1, -1) if i == 0 else (2 * i - 1, 2 * i - 1))]

    made = engine.generate_drafted(prompt, drafter, 40, eos_id=None)
    assert len(made.token_ids) == 40 and engine.cache.free_pages() == engine.cache.total_pages()
    if dtype == torch.float32 and cache_dtype == "auto":  # (16 bits and numbers next to a border leave the arg-max alone only mostly)
        assert made.token_ids == answer and made.steps <= 8
