"""Rows into caches of every type and back, against 64 bits: the write, the read, what they leave alone."""

from __future__ import annotations

import pytest
import torch

from distie_b200.kernels import RotaryTable
from plain_cached import E4M3, Case, finish, half_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def sets():
    from distie_b200.kernels import make_kernels

    return {dtype: make_kernels(dtype, DEV) for dtype in (BF16, F32)}


def rotary(n, interleaved=False, factor=1.0, theta=1e4):
    return RotaryTable((theta ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)).float().to(DEV), n, interleaved, factor)


def check_rows(case, which, want, request_rows):
    """The stored rows of the new tokens against 64-bit ones; every other row of the pool as it was before."""
    place = [(int(case.table[case.seats[r], slot // case.page]), slot % case.page) for r, slot in request_rows]
    pages, at = torch.tensor([p for p, _ in place]), torch.tensor([a for _, a in place])
    got = case.rows(which)[pages, :, at]
    most = want.abs().amax(-1, keepdim=True)
    # float32 sums, a root, a rotation: some 2^-21 of the row's largest; then half a step of the cache's type.
    slack = 2.0**-20 * most
    if case.kv.k.dtype == E4M3:
        scale = getattr(case.kv, which + "_scale").double().cpu()[pages, :, at]
        torch.testing.assert_close(scale, most[..., 0] / 448.0, rtol=2.0**-20, atol=0.0)
        slack = slack + torch.maximum(half_step(E4M3) * want.abs(), 2.0**-10 * most / 448.0)
    else:
        slack = slack + half_step(case.kv.k.dtype) * want.abs()
    assert bool(((got - want).abs() <= slack).all()), float(((got - want).abs() - slack).max())
    return pages, at


WRITES = [
    # heads, kv heads, key size, value size, rotary (size, interleaved, factor), norm mode, weights, bias, slices, page, q_temp
    (12, 2, 128, 128, (128, False, 1.0), 0, False, True, 1, 16, None),
    (12, 2, 128, 128, (128, False, 1.0), 1, True, True, 3, 16, (0.1, 64.0)),
    (4, 4, 64, 64, (64, False, 1.2), 1, False, False, 2, 32, None),
    (5, 5, 48, 48, (32, True, 1.0), 1, True, True, 1, 5, None),
    (8, 1, 64, 64, (32, False, 1.0), 0, False, True, 1, 8, None),
    (6, 3, 16, 40, None, 0, False, False, 4, 4, None),
    (2, 1, 256, 256, (256, True, 1.0), 0, False, True, 1, 16, None),
    (3, 3, 33, 7, None, 1, True, True, 2, 3, None),
]


@pytest.mark.parametrize("cache", ["e4m3", "typed"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("w", range(len(WRITES)))
def test_projection_into_the_cache(sets, dtype, cache, w):
    heads, kv, dim, vdim, turn, mode, weighted, biased, slices, page, temp = WRITES[w]
    k = sets[dtype]
    # A tree, a chain of one and a long one far into a request: places that differ from positions.
    case = Case("tree", [(7, [-1, 0, 0, 1, -1]), (0, [-1]), (3001, list(range(-1, 40)))], kv, dim, vdim, page, E4M3 if cache == "e4m3" else dtype,
                dtype, DEV, seed=w)
    before = {n: case.rows(n) for n in "kv"}
    g = torch.Generator().manual_seed(100 + w)
    columns = (heads + kv) * dim + kv * vdim
    proj = torch.randn(slices, case.step.num_tokens, columns + 8, generator=g).to(DEV)[..., :columns]
    bias = torch.randn(columns, generator=g).to(DEV) if biased else None
    weights = [(1 + 0.2 * torch.randn(dim, generator=g)).to(DEV) if weighted else None for _ in range(2)]
    table = rotary(*turn) if turn else None
    q = torch.zeros((case.step.num_tokens, heads * dim), dtype=dtype, device=DEV)
    k.qkv_norm_write(proj, bias, case.step, case.kv, table, heads, kv, dim, vdim, 1e-6 if mode else None, *weights, temp, q)
    k.check_errors()
    want = finish(proj, case.positions, heads, kv, dim, vdim, bias, table, (mode, 1e-6, *weights) if mode else None, temp)
    most = want[0].abs().amax(-1, keepdim=True)
    off = (q.double().cpu().reshape(want[0].shape) - want[0]).abs()
    assert bool((off <= 2.0**-20 * most + half_step(dtype) * want[0].abs()).all())
    requests = [r for r, n in enumerate(case.news) for _ in range(n)]
    for which, rows in (("k", want[1]), ("v", want[2])):
        pages, at = check_rows(case, which, rows, list(zip(requests, case.slots)))
        after, held = case.rows(which), before[which]
        after[pages, :, at] = held[pages, :, at]
        assert torch.equal(after, held)  # nothing else was touched


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_every_write_goes_to_an_8_bit_cache(sets, dtype):
    """rope_kv_write (slices, and a finished projection in place), qkv_rope_write, kv_write and the keys that are values."""
    k, heads, kv, dim = sets[dtype], 4, 2, 64
    g = torch.Generator().manual_seed(3)
    requests = [(5, 1), (130, 1), (17, 6), (0, 140)]
    columns = (heads + 2 * kv) * dim
    where = lambda case: [(r, s) for (r, s) in zip([r for r, n in enumerate(case.news) for _ in range(n)], case.slots)]  # noqa: E731
    new = lambda: Case("portion", requests, kv, dim, dim, 16, E4M3, dtype, DEV, seed=1)  # noqa: E731
    case = new()
    bias, table, tokens = torch.randn(columns, generator=g).to(DEV), rotary(dim), case.step.num_tokens
    proj = torch.randn(2, tokens, columns, generator=g).to(DEV)
    q = torch.empty((tokens, heads * dim), dtype=dtype, device=DEV)
    k.rope_kv_write(proj, case.step, case.kv, table, heads, kv, dim, bias=bias, q_out=q)
    want = finish(proj, case.positions, heads, kv, dim, dim, bias, table)
    check_rows(case, "k", want[1], where(case))
    check_rows(case, "v", want[2], where(case))
    near = lambda a, b: bool(((a.double().cpu().reshape(b.shape) - b).abs() <= 2.0**-20 * b.abs().amax(-1, keepdim=True) + half_step(dtype) * b.abs()).all())  # noqa: E731
    assert near(q, want[0])
    case, typed = new(), proj.sum(0).to(dtype)  # a finished projection: q is turned in place
    held = typed.clone()
    k.rope_kv_write(held, case.step, case.kv, table, heads, kv, dim, q_out=q)
    want = finish(typed, case.positions, heads, kv, dim, dim, None, table)
    check_rows(case, "k", want[1], where(case))
    check_rows(case, "v", want[2], where(case))
    assert near(q, want[0]) and torch.equal(q, held[:, : heads * dim]) and torch.equal(held[:, heads * dim :], typed[:, heads * dim :])
    case = new()
    k.kv_write(typed[:, heads * dim : (heads + kv) * dim], typed[:, (heads + kv) * dim :], case.step, case.kv)
    want = finish(typed, case.positions, heads, kv, dim, dim)
    check_rows(case, "k", want[1], where(case))
    check_rows(case, "v", want[2], where(case))
    for eps in (None, 1e-5):
        case, shared = new(), proj[..., : (heads + kv) * dim]
        k.qk_rope_norm_write(shared, bias[: (heads + kv) * dim], case.step, case.kv, table, heads, kv, dim, eps, q)
        want = finish(shared, case.positions, heads, kv, dim, dim, bias[: (heads + kv) * dim], table, None if eps is None else (2, eps, None, None), values=False)
        check_rows(case, "k", want[1], where(case))
        check_rows(case, "v", want[2], where(case))
        assert near(q, want[0])
    k.check_errors()


def test_far_positions_turn_exactly(sets):
    """An angle of many turns: the rounding of position * frequency, 4e-3 at 100,000, does not reach the rows."""
    k = sets[F32]
    case = Case("single", [(100003, 1), (65537, 1), (1, 1)], 1, 64, 64, 16, F32, F32, DEV)
    case.step.slots = torch.tensor(case.slots, dtype=torch.int32, device=DEV)  # (an engine's own rows take the plain kernel)
    proj, table = torch.randn(1, 3, 3 * 64, generator=torch.Generator().manual_seed(5)).to(DEV), rotary(64)
    q = torch.empty((3, 64), device=DEV)
    k.qkv_norm_write(proj, None, case.step, case.kv, table, 1, 1, 64, 64, None, None, None, None, q)
    want = finish(proj, case.positions, 1, 1, 64, 64, None, table)[0][:, 0]
    # cos and sin to 2 ulp, products and their sum: below 2^-21 of the row's largest.
    assert bool(((q.double().cpu() - want).abs() <= 2.0**-20 * want.abs().amax(-1, keepdim=True)).all())


def test_rows_that_are_not_finite_and_rows_of_zeros(sets):
    k = sets[BF16]
    case = Case("tree", [(20, [-1, 0, 1, 2])], 2, 64, 64, 16, E4M3, BF16, DEV)
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1))
    x[0, 1, 5], x[1, 0, 63], x[2, 1] = float("nan"), float("-inf"), 0.0
    x[3, 0] *= 1e-38 / x[3, 0].abs().max()
    flat = x.reshape(4, 128).to(DEV)
    k.kv_write(flat, flat, case.step, case.kv)
    rows = case.held("k", 0)[:, 20:].transpose(0, 1)
    bad = torch.zeros(4, 2, dtype=torch.bool)
    bad[0, 1] = bad[1, 0] = True
    assert bool(rows[bad].isnan().all()) and bool(torch.isfinite(rows[~bad]).all())
    assert bool((rows[2, 1] == 0).all())
    # A row whose scale is a subnormal number (2^-149 steps): the scale is off by half a step of its own, the number by half of one.
    tiny = x[3, 0].double()
    assert bool(((rows[3, 0] - tiny).abs() <= 2.0**-4 * tiny.abs() + 448 * 2.0**-149 + 2.0**-10 * 1e-38 / 448).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dims", [(128, 128, 16, 4), (64, 64, 8, 2), (48, 40, 5, 3), (20, 20, 16, 1)])
def test_pages_read_back(sets, dtype, dims):
    dim, vdim, page, kv = dims
    k = sets[dtype]
    case = Case("portion", [(9, 1), (40, 1), (0, 2), (333, 71), (page, page), (2 * page - 1, 2)], kv, dim, vdim, page, E4M3, dtype, DEV, seed=7)
    read = k.kv_read(case.step, case.kv)
    k.check_errors()
    assert read.k.dtype == dtype and read.num_pages == read.k.shape[0]
    at = 0
    for r, (past, new) in enumerate(zip(case.pasts, case.news)):
        if new == 1:
            continue
        count = -(-(past + new) // page)
        row = read.block_table[case.seats[r]].tolist()
        assert row[:count] == list(range(at, at + count)) and all(c == -1 for c in row[count:])
        for which in "kv":
            got = getattr(read, which)[at : at + count].transpose(0, 1).reshape(kv, count * page, -1).double().cpu()
            want = case.held(which, r).float().to(dtype).double()  # a product of two float32 numbers, rounded twice at most
            assert bool(((got[:, : past + new] - case.held(which, r)).abs() <= (half_step(dtype) + 2.0**-24) * case.held(which, r).abs()).all())
            assert torch.equal(got[:, : past + new], want) or dtype == BF16
            assert bool((got[:, past + new :] == 0).all())
        at += count
    assert at == read.num_pages


@pytest.mark.parametrize("what", [dict(window=30), dict(chunk=64), dict(window=30, keep_first=20)])
def test_pages_behind_a_window_are_left_out(sets, what):
    k, page = sets[BF16], 8
    case = Case("portion", [(100, 5), (3, 9), (200, 40)], 2, 64, 64, page, E4M3, BF16, DEV, seed=2)
    held = {r: torch.stack([case.held("k", r), case.held("v", r)]) for r in range(3)}
    needed = {}
    for r, past in enumerate(case.pasts):  # a cache gives the pages back that no later token sees
        first = max(0, past - what["window"] + 1) if what.get("window") else past // what["chunk"] * what["chunk"]
        kept = -(-what.get("keep_first", 0) // page)
        for c in range(-(-(past + case.news[r]) // page)):
            if kept <= c < first // page:
                case.kv.block_table[case.seats[r], c] = -1
            else:
                needed.setdefault(r, []).append(c)
    read = k.kv_read(case.step, case.kv, **what)
    k.check_errors()
    for r, columns in needed.items():
        ids = read.block_table[case.seats[r]].long().cpu()
        assert [c for c in range(ids.numel()) if ids[c] >= 0] == columns
        for n, pages in enumerate((read.k, read.v)):
            got = pages[ids[columns]].double().cpu().transpose(0, 1)
            for i, c in enumerate(columns):
                want = held[r][n][:, c * page : (c + 1) * page]
                assert bool(((got[:, i, : want.shape[1]] - want).abs() <= 2.0**-7 * want.abs()).all())


def test_pages_that_are_missing_are_reported(sets):
    from distie_b200.kernels.library import KernelError

    k = sets[BF16]
    case = Case("tree", [(20, [-1, 0, 1]), (3, [-1])], 2, 64, 64, 16, E4M3, BF16, DEV)
    case.kv.block_table[case.seats[0], 1] = -1
    rows = torch.randn(4, 128, device=DEV)
    before = case.kv.k.float().clone()
    k.kv_write(rows, rows, case.step, case.kv)
    with pytest.raises(KernelError, match="missing from its block table"):
        k.check_errors()
    changed = (case.kv.k.float() != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(case.table[case.seats[1], 0])]  # the other request's row is where it belongs
    case = Case("portion", [(20, 4)], 2, 64, 64, 16, E4M3, BF16, DEV)
    case.kv.block_table[case.seats[0], 0] = case.kv.num_pages
    k.kv_read(case.step, case.kv)
    with pytest.raises(KernelError, match="does not cover"):
        k.check_errors()
