"""One rotation: rows of drafted tokens, of 8-bit caches and of every other step agree however far they stand."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from distie_b200.config import EngineConfig, get_architecture
from distie_b200.config.model_spec import PartSpec
from distie_b200.engine.batch import BatchEntry
from distie_b200.engine.engine import Engine
from distie_b200.kernels import make_kernels
from distie_b200.parts.base import POSITION_ENCODINGS
from plain_cached import E4M3, Case
from test_cached_rows_gpu import BF16, DEV, F32

import helpers

pytestmark = pytest.mark.gpu
FAR = [(65537, 1), (100003, 1), (7, 1), (30000, 1)]


@pytest.fixture(scope="module")
def sets():
    return {dtype: make_kernels(dtype, DEV) for dtype in (BF16, F32)}


def new_rows(pages, table, places, page):
    """The rows at the places of a request, [places, kv heads, size]."""
    return torch.stack([pages[int(table[p // page]), :, p % page] for p in places]).double()


def engine_table(**params):
    """The rotary table as a model's layers are built with."""
    return POSITION_ENCODINGS.get("rotary").build(PartSpec("rotary", params=params), SimpleNamespace(device=torch.device(DEV))).rotary_table()


ENCODINGS = [(128, dict(head_dim=128, theta=1e6)), (64, dict(head_dim=64, theta=1e4, factor=1.25)), (48, dict(head_dim=48, theta=5e4, rotary_dim=32)),
             (64, dict(head_dim=64, theta=1e4, interleaved=True))]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim, params", ENCODINGS)
def test_rows_at_places_are_the_rows_of_other_steps(sets, dtype, dim, params):
    """The same projection written by a step whose tokens stand at their positions and by one that gives their places."""
    k, heads, kv, table = sets[dtype], 2, 1, engine_table(**params)
    columns = (heads + 2 * kv) * dim
    proj = torch.randn(2, len(FAR), columns, generator=torch.Generator().manual_seed(1)).to(DEV)
    bias = torch.randn(columns, generator=torch.Generator().manual_seed(2)).to(DEV)
    made = []
    for apart in (False, True):
        case = Case("single", FAR, kv, dim, dim, 16, dtype, dtype, DEV)
        rows = lambda pages: torch.cat([new_rows(pages, case.table[case.seats[r]], [p], 16) for r, (p, _) in enumerate(FAR)])  # noqa: E731
        if apart:
            case.step.slots = torch.tensor(case.slots, dtype=torch.int32, device=DEV)
        q = torch.empty((len(FAR), heads * dim), dtype=dtype, device=DEV)
        k.rope_kv_write(proj, case.step, case.kv, table, heads, kv, dim, bias=bias, q_out=q)
        made.append([q.clone(), rows(case.kv.k), rows(case.kv.v)])
        k.qkv_norm_write(proj, bias, case.step, case.kv, table, heads, kv, dim, dim, 1e-6, None, None, None, q)
        made[-1] += [q, rows(case.kv.k)]
    k.check_errors()
    # A rotation of part of a head, or of neighbours, is no kernel's of the ordinary bfloat16 steps: there rope_kv_write rounds the
    # projection to bfloat16 before it turns it.  A pair (a, b) is then off by 2^-8 of each, its rotation by up to
    # 2^-8 (|a cos| + |b sin|) <= 2^-8 sqrt(a^2 + b^2) <= 2^-8 sqrt(2) of the row's largest turned number, less than 2^-7 of it.
    twice = dtype == BF16 and (params.get("interleaved") or params.get("rotary_dim", dim) < dim)
    for i, (one, other) in enumerate(zip(*made)):
        one, other = (x.double().reshape(len(FAR), -1, dim) for x in (one, other))
        most = one.abs().amax(-1, keepdim=True)
        # The same angles, sums of two products in float32: a few 2^-24 of the row's largest, then half a step of the type where the two
        # sides fall apart (bfloat16: a whole step).
        slack = 2.0**-21 * most + (2.0**-7 * one.abs() if dtype == BF16 else 0.0) + (2.0**-7 * most if twice and i < 3 else 0.0)
        assert bool(((one - other).abs() <= slack).all()), float((one - other).abs().max())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_over_the_8_bit_cache_of_another_layer(sets, dtype):
    """A layer that reads another layer's cache writes none: its queries turn as those of the layer that writes it."""
    k, heads, kv, dim = sets[dtype], 2, 1, 64
    table = engine_table(head_dim=dim, theta=1e4)
    case = Case("single", FAR, kv, dim, dim, 16, E4M3, dtype, DEV)
    proj = torch.randn(1, len(FAR), (heads + 2 * kv) * dim, generator=torch.Generator().manual_seed(3)).to(DEV)
    own, borrowed = (torch.empty((len(FAR), heads * dim), dtype=dtype, device=DEV) for _ in range(2))
    k.rope_kv_write(proj, case.step, case.kv, table, heads, kv, dim, q_out=own)
    k.rope_kv_write(proj, case.step, None, table, heads, kv, dim, q_out=borrowed)
    k.check_errors()
    most = own.double().abs().reshape(-1, dim).amax(-1).repeat_interleave(dim).reshape(own.shape)
    off = (own.double() - borrowed.double()).abs()
    assert bool((off <= 2.0**-21 * most + (2.0**-7 * own.double().abs() if dtype == BF16 else 0.0)).all()), float(off.max())


@pytest.mark.parametrize("past", [30000, 65000])
def test_a_far_chain_leaves_the_rows_of_single_steps(past):
    """A chain of drafted tokens behind a long past, and the same tokens one by one: the rows that both leave in the cache."""
    cfg, page, weights = helpers.tiny("D")
    cfg["max_position_embeddings"] = past + 64
    arch = get_architecture(cfg["architectures"][0])
    config = EngineConfig(num_blocks=2 * (past + 64) // page + 4, page_size=page, max_seqs=2, token_budget=64, dtype="float32", device=DEV,
                          decode_graphs=False)
    engine = Engine.assemble(arch, arch.config_cls.from_dict(cfg), weights, make_kernels(F32, DEV), config)
    seats = [engine.cache.open_seat() for _ in range(2)]
    for seat in seats:
        assert engine.cache.grow(seat, past + 12)
    draft = helpers.random_ids(cfg["vocab_size"], 12, 4)
    engine.runner.step([BatchEntry(seats[0], draft, past, (0,), list(range(-1, 11)))])
    for i, token in enumerate(draft):
        engine.runner.step([BatchEntry(seats[1], [token], past + i, (0,))])
    engine.runner.finish_step()
    for group in engine.cache.groups:
        for slot in group.slots:
            one, other = (new_rows(engine.cache.kv_slot(slot).k, group.host_table[s], range(past, past + 12), page) for s in seats)
            # The orders of float32 sums differ, 2^-18 or so behind some layers of a thousand terms.  An angle of 30,000 radians that is
            # rounded is off by up to 2^-10, one of 65,000 by 2^-9, and so is the row.
            assert float((one - other).abs().max()) <= 2.0**-13 * float(other.abs().max())


def test_exact_angles_up_to_their_bound(sets):
    """Without ``rounded`` the angle is the exact product: its rounding error goes back in as a small rotation, good to 2^18."""
    from plain_cached import finish
    from test_cached_rows_gpu import rotary

    requests = [(2**18 - 1, 1), (2**18 - 5, 1)]
    case = Case("single", requests, 1, 64, 64, 16, F32, F32, DEV)
    case.step.slots = torch.tensor(case.slots, dtype=torch.int32, device=DEV)
    proj = torch.randn(1, 2, 3 * 64, generator=torch.Generator().manual_seed(5)).to(DEV)
    q = torch.empty((2, 64), device=DEV)
    sets[F32].qkv_norm_write(proj, None, case.step, case.kv, rotary(64), 1, 1, 64, 64, None, None, None, None, q)
    want = finish(proj, case.positions, 1, 1, 64, 64, None, rotary(64))[0][:, 0]
    # cos and sin to 2 ulp, what the correction leaves out (2^-7 cubed over 6: 2^-23.6), products and their sum.
    assert bool(((q.double().cpu() - want).abs() <= 2.0**-20 * want.abs().amax(-1, keepdim=True)).all())
