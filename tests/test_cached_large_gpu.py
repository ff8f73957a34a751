"""Caches whose offsets pass 32 bits, and steps of many portions: the same results, to the bit, as small ones give."""

from __future__ import annotations

import pytest
import torch

from distie_b200.kernels import make_kernels
from distie_b200.kernels.interface import KvSlot
from plain_cached import E4M3, Case
from test_cached_attention_gpu import BF16, DEV, F32, queries

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sets():
    return {dtype: make_kernels(dtype, DEV) for dtype in (BF16, F32)}


def moved(case, elements):
    """The case's pages as the last ones of a pool whose keys alone are more than ``elements`` elements."""
    kv = case.kv
    per_page = kv.k[0].numel()
    pages = elements // per_page + kv.num_pages + 1
    first = pages - kv.num_pages

    def large(rows):
        if rows is None:
            return None
        out = torch.empty((pages, *rows.shape[1:]), dtype=rows.dtype, device=DEV)
        held = out.view(torch.uint8) if rows.dtype == E4M3 else out
        held[first:] = rows.view(torch.uint8) if rows.dtype == E4M3 else rows
        return out

    table = torch.where(kv.block_table >= 0, kv.block_table + first, kv.block_table)
    return KvSlot(large(kv.k), large(kv.v), table, kv.page_size, pages, large(kv.k_scale), large(kv.v_scale)), first


@pytest.mark.parametrize("kind, cache, dtype, dim", [
    ("single", E4M3, BF16, 128), ("single", E4M3, F32, 64), ("tree", E4M3, BF16, 64), ("tree", BF16, BF16, 128), ("tree", F32, F32, 48),
])
def test_offsets_beyond_32_bits(sets, kind, cache, dtype, dim):
    k, heads = sets[dtype], 6
    requests = [(300, 1), (17, 1)] if kind == "single" else [(300, [-1, 0, 0]), (17, [-1, 0])]
    case = Case(kind, requests, 2, dim, dim, 16, cache, dtype, DEV)
    slot, first = moved(case, 2**31 + 2**20)
    g = torch.Generator().manual_seed(4)
    rows = torch.randn(2, case.step.num_tokens, 2 * dim, generator=g).to(dtype).to(DEV)
    q, outs = queries(case, heads, dtype), []
    for kv in (case.kv, slot):
        k.kv_write(rows[0], rows[1], case.step, kv)
        out = torch.empty((case.step.num_tokens, heads * dim), dtype=dtype, device=DEV)
        k.attention(q, out, case.step, kv, heads, 2, dim, None, dim**-0.5)
        outs.append(out)
    k.check_errors()
    assert torch.equal(outs[0], outs[1])
    for which in ("k", "v", "k_scale", "v_scale"):
        small, large = getattr(case.kv, which), getattr(slot, which)
        if small is not None:
            assert torch.equal(small.view(torch.uint8), large[first:].contiguous().view(torch.uint8))


@pytest.mark.parametrize("portions", [8, 9, 256, 257, 300])
def test_many_portions_are_read_back(sets, portions):
    case = Case("portion", [(7, 1), *((r % 23, 2 + r % 5) for r in range(portions))], 1, 16, 16, 4, E4M3, BF16, DEV)
    read = sets[BF16].kv_read(case.step, case.kv)
    sets[BF16].check_errors()
    at = 0
    for r, (past, new) in enumerate(zip(case.pasts, case.news)):
        if new == 1:
            continue
        count = -(-(past + new) // 4)
        assert read.block_table[case.seats[r]].tolist()[:count] == list(range(at, at + count))
        for which in "kv":
            got = getattr(read, which)[at : at + count].transpose(0, 1).reshape(1, count * 4, 16).double().cpu()
            want = case.held(which, r)  # float32 product, rounded to bfloat16
            assert bool(((got[:, : past + new] - want).abs() <= (2.0**-8 + 2.0**-24) * want.abs() * (1 + 2.0**-8)).all())
            assert bool((got[:, past + new :] == 0).all())
        at += count
    assert at == read.num_pages
