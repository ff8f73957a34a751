"""Prompt attention over 8-bit caches: the pages read back and the table that names them, however busy the GPU is."""

from __future__ import annotations

from dataclasses import replace

import pytest
import torch

from distie_b200.kernels import make_kernels
from plain_cached import E4M3, Case, half_step
from test_cached_attention_gpu import BF16, DEV, F32, queries

pytestmark = pytest.mark.gpu

# Steps one after another (single tokens first, as every step has them): what a step's table held is wrong for the next one.
SHORT = [[(40, 1), (0, 200), (301, 130)], [(7, 30), (513, 64), (90, 3)], [(3, 1), (0, 5), (260, 140), (17, 33)], [(301, 130), (0, 200)]]
LONG = [[(12, 1), (6000, 130)], [(5, 1), (5500, 257)], [(3100, 70), (4200, 140)]]


@pytest.fixture(scope="module")
def sets():
    return {dtype: make_kernels(dtype, DEV) for dtype in (BF16, F32)}


def exact_case(requests, kv, dim, dtype, seed):
    """A case whose rows come back exactly: e4m3 numbers times a power of two are bfloat16 numbers."""
    case = Case("portion", requests, kv, dim, dim, 16, E4M3, dtype, DEV, seed=seed)
    case.masks = [torch.ones(n, n).tril().bool() for n in case.news]
    case.kv.k_scale.fill_(2.0**-7)
    case.kv.v_scale.fill_(2.0**-7)
    return case


def other_ids(case, pages):
    """Memory of the size of the case's block table, as the next allocation finds it: other page ids, all of them valid."""
    g = torch.Generator().manual_seed(5)
    held = [torch.randint(0, pages, case.table.shape, dtype=torch.int32, generator=g).to(DEV) for _ in range(4)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("dtype, dim, heads, kv, steps, kernel", [
    (BF16, 128, 12, 2, SHORT, "attention_prefill_tcgen05"), (BF16, 64, 8, 2, SHORT, "attention_prefill_tcgen05"),
    (BF16, 128, 12, 2, LONG, "attention_prefill_pairs"), (BF16, 64, 24, 2, LONG, "attention_prefill_pairs"),
    (BF16, 48, 4, 2, SHORT, "attention_prefill_tcgen05"), (F32, 64, 8, 2, SHORT, "rows_read"),
])
def test_prompt_attention_while_the_gpu_is_busy(sets, dtype, dim, heads, kv, steps, kernel):
    """The launches of a step stand behind queued work, so that they start as early as they may; the portions change from step to
    step, and the memory of the table holds other ids."""
    k = sets[dtype]
    cases = [exact_case(requests, kv, dim, dtype, seed) for seed, requests in enumerate(steps)]
    pages = min(sum(-(-(p + n) // 16) for p, n in zip(c.pasts, c.news) if n > 1) for c in cases)
    qs = [queries(c, heads, dtype, seed=20 + i) for i, c in enumerate(cases)]
    a = torch.randn(4096, 4096, dtype=BF16, device=DEV)
    before = k.kernel_counts.get(kernel, 0)
    for what in ({}, dict(window=200)):
        outs = [torch.empty_like(q) for q in qs]
        for case, q, out in zip(cases, qs, outs):
            other_ids(case, pages)
            case.step = replace(case.step, derived={})
            for _ in range(12):
                a @ a
            rows = torch.randn(case.step.num_tokens, 2 * kv * dim, device=DEV).to(E4M3).float() * 2.0**-7  # what the step writes first
            rows[:, ::dim] = 448.0 * 2.0**-7  # (the largest of every row: its scale is 2^-7 too)
            k.kv_write(rows[:, : kv * dim], rows[:, kv * dim :], case.step, case.kv)
            for _ in range(2):  # layers of a step share its table
                k.attention(q, out, case.step, case.kv, heads, kv, dim, what.get("window"), dim**-0.5)
        torch.cuda.synchronize()
        k.check_errors()
        for case, q, out in zip(cases, qs, outs):
            calm = torch.empty_like(out)
            k.attention(q, calm, replace(case.step, derived={}), case.kv, heads, kv, dim, what.get("window"), dim**-0.5)
            torch.cuda.synchronize()
            assert torch.equal(out, calm)
            want, size = case.attention(q, heads, dim**-0.5, **what)
            # Rounded are the weights (of the prompt kernels and of single tokens) and the output; float32 sums and exponentials of scores
            # up to 2^5 are off by 2^-15.
            slack = half_step(dtype) * want.abs() + ((half_step(BF16) if dtype == BF16 else 0.0) + 2.0**-15) * size
            slack = slack + 2 * 2.0**-20 * case.reach(q, heads, dim**-0.5) * size + (case.least if dtype == BF16 else 0.0)
            assert bool(((out.double().cpu() - want).abs() <= slack).all()), float(((out.double().cpu() - want).abs() - slack).max())
    assert k.kernel_counts[kernel] > before


def test_a_captured_step_reads_the_pages_of_other_seats(sets):
    """A step with portions replayed after its requests moved to other seats: the table of the pages read back follows."""
    k, dim, heads, kv = sets[BF16], 64, 4, 2
    case = exact_case([(20, 30), (0, 50)], kv, dim, BF16, 3)
    q = queries(case, heads, BF16)
    out = torch.empty_like(q)
    call = lambda: k.attention(q, out, case.step, case.kv, heads, kv, dim, None, dim**-0.5)  # noqa: E731
    call()
    alone = out.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    spare = next(s for s in range(case.table.shape[0]) if s not in case.seats)
    case.kv.block_table[spare] = case.kv.block_table[case.seats[0]]
    case.kv.block_table[case.seats[0]] = -1
    case.step.seq_seat[0] = spare
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        k.check_errors()
        assert torch.equal(out, alone)
