"""Drafted generation beside other requests, near its end, and with drafters that are wrong."""

from __future__ import annotations

import pytest
import torch

import helpers
import test_fovudra as fovudra
from ref_cached import RefCached
from test_cached_engine import engine_for

from distie_b200.cache import CacheManager
from distie_b200.parts.base import CacheNeed

NONE = lambda ids: ([], [])  # noqa: E731


@pytest.mark.parametrize("budget", [4096, 8])
def test_pages_behind_a_window_go_back_before_the_first_guess(budget):
    """Layers with a window of 8 over pages of 4: behind a prompt of 32 tokens they hold three pages, not eight, and the request
    goes on beside another one that holds the last."""
    layer = fovudra._attention(4, 2, 16, 8, 0, 16, 1e4, None, 0.25, fovudra._moe(3, 1, 20, None))
    cfg = {"architecture": "Fovudra", "vocab": 101, "width": 48, "norm": {"eps": 1e-5}, "layers": [layer, layer]}
    weights = fovudra.pf.random_weights(cfg, 5)
    prompt = helpers.random_ids(101, 32, 8)
    made = []
    for drafted in (False, True):
        engine = fovudra.engine_of(cfg, weights, 4, RefCached(torch.float32), 9, token_budget=budget, max_model_len=40)
        other = engine.cache.open_seat()
        assert engine.cache.grow(other, 1)
        if drafted:
            made.append(engine.generate_drafted(prompt, NONE, 4, eos_id=None).token_ids)
        else:
            made.append(engine.generate([prompt], max_new_tokens=4, ignore_eos=True)[0].token_ids)
        engine.cache.close_seat(other)
        assert engine.cache.free_pages() == engine.cache.total_pages()
    assert made[0] == made[1] and len(made[0]) == 4


@pytest.mark.parametrize("parents, word", [([-2], "parent"), ([-1, -2, 0], "parent"), ([-1, 1], "parent"), ([-1] * 300 + [300], "parent")])
def test_parents_that_are_none_are_refused(parents, word):
    """-2 is no parent: as the number behind the last token's it would have been taken for a second root.  The guesses that a step
    has no room for are looked at too."""
    engine, _, _ = engine_for("A")
    with pytest.raises(ValueError, match=word):
        engine.generate_drafted([1, 2], lambda ids: ([5] * len(parents), parents), 40, eos_id=None)
    assert engine.cache.free_pages() == engine.cache.total_pages() and engine.cache.free_seats == 8


def checked(engine):
    """The numbers of guesses that each step of an engine brings."""
    seen, run = [], engine.runner.step

    def step(entries):
        if entries[0].parents is not None:
            seen.append(len(entries[0].tokens) - 1)
        return run(entries)

    engine.runner.step = step
    return seen


def test_guesses_that_the_request_has_no_use_for_are_not_checked():
    """With n tokens still wanted behind the one that a step begins with, guesses below depth n - 1 cannot become output."""
    engine, cfg, _ = engine_for("A")
    prompt, vocab = helpers.random_ids(cfg["vocab_size"], 9, 3), cfg["vocab_size"]
    answer = engine.generate([prompt], max_new_tokens=12, ignore_eos=True)[0].token_ids

    def drafter(ids):  # a chain of five right guesses, and two wrong ones beside its second and at its end
        at = len(ids) - len(prompt)
        right = (answer + answer)[at : at + 5]
        return [*right[:2], (right[1] + 1) % vocab, *right[2:], (right[4] + 1) % vocab], [-1, 0, 0, 1, 3, 4, 4]

    seen = checked(engine)
    made = engine.generate_drafted(prompt, drafter, 9, eos_id=None)
    # Nine tokens: the prompt's, five guesses and the one behind them, then two more, of which one can be a guess.
    assert made.token_ids == answer[:9] and seen == [7, 1] and made.drafted == 8 and made.accepted == 6
    engine, _, _ = engine_for("A")
    seen = checked(engine)
    made = engine.generate_drafted(prompt, lambda ids: ([answer[len(ids) - len(prompt)]] * 300, [-1] * 300), 2, eos_id=None)
    assert made.token_ids == answer[:2] and seen == [0] and made.drafted == 0


def test_a_refused_path_moves_nothing():
    """A group whose window has given a place's page back refuses the path; no other group has moved its rows then."""
    needs = {0: CacheNeed(1, 8), 1: CacheNeed(1, 8, window=4)}
    cache = CacheManager(needs, num_pages=8, page_size=2, max_seats=1, max_tokens_per_request=16, dtype=torch.float32, device="cpu")
    seat = cache.open_seat()
    assert cache.grow(seat, 12)
    for slot in (0, 1):
        cache.kv_slot(slot).k.copy_(torch.arange(cache.kv_slot(slot).k.numel()).reshape(cache.kv_slot(slot).k.shape))
    cache.trim(seat, 12)  # (as if all twelve had been kept)
    before = [cache.kv_slot(slot).k.clone() for slot in (0, 1)]
    with pytest.raises(ValueError, match="holds no page"):
        cache.keep_places(seat, 4, [1, 3])
    assert all(torch.equal(cache.kv_slot(slot).k, old) for slot, old in zip((0, 1), before))
