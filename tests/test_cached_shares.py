"""Shares of the keys: what a step of a new length costs the host."""

from __future__ import annotations

import pytest
import torch

from distie_b200.kernels import cached
from distie_b200.kernels.cached import decode_splits, rows_splits
from distie_b200.kernels.interface import E4M3, KvSlot
from test_cached_refusals import Checks, step


@pytest.mark.parametrize("dim, rule, launched", [(64, decode_splits, "distie_attention_decode_e4m3"), (32, rows_splits, "distie_attention_rows")])
def test_a_step_one_key_longer_does_not_search_again(monkeypatch, dim, rule, launched):
    names = []
    monkeypatch.setattr(cached, "packed", lambda name: (lambda block: names.append(name) or 0, lambda *args: args))
    shape, lengths = (2, 2, 16), range(4001, 4321)
    slot = KvSlot(torch.zeros(*shape, dim).to(E4M3), torch.zeros(*shape, dim).to(E4M3), torch.zeros(2, 4, dtype=torch.int32), 16, 2,
                  torch.ones(shape), torch.ones(shape))
    rows = torch.zeros(3, 6 * dim, dtype=torch.bfloat16)
    before = rule.cache_info().misses
    for length in lengths:
        s = step(max_kv_len=length)
        Checks()._attention_rows(rows, torch.zeros_like(rows), s, slot, 6, 2, dim, 0, 0, 1.0, 0, 0.0, None, 3, 3)
    assert names == [launched] * len(lengths)
    assert rule.cache_info().misses - before <= len(lengths) // 32 + 1
