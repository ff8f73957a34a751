"""Attention over 8-bit caches and of drafted tokens over caches of every type, against 64 bits."""

from __future__ import annotations

import pytest
import torch

from plain_cached import E4M3, Case, half_step, random_parents

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def sets():
    from distie_b200.kernels import make_kernels

    return {dtype: make_kernels(dtype, DEV) for dtype in (BF16, F32)}


def queries(case, heads, dtype, seed=9, pad=0):
    g = torch.Generator().manual_seed(seed)
    return (1.5 * torch.randn(case.step.num_tokens, heads * case.dim + pad, generator=g)).to(dtype).to(DEV)


def check(k, case, heads, q=None, large=False, tiny=0.0, **what):
    dtype = k.dtype
    q = queries(case, heads, dtype) if q is None else q
    out = torch.full((case.step.num_tokens, heads * case.value_dim), 7.0, dtype=dtype, device=DEV)
    scale = case.dim**-0.5
    sink = what.get("sink")
    k.attention(q, out, case.step, case.kv, heads, case.kv_heads, case.dim, what.get("window"), scale, what.get("chunk"),
                what.get("keep_first", 0), what.get("softcap", 0.0), sink)
    k.check_errors()
    want, size = case.attention(q, heads, scale, **what)
    got = out.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), "not-a-number where it does not belong, or none where it does"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    # The output's rounding, relative to it; the rounding of the softmax's weights to 16 bits where products take them
    # (relative to the sum of weight times magnitude; the sum that divides them is not rounded), and float32 sums and exponentials: scores
    # of up to 50 are off by 50 * 2^-22 or so, and so are their exponentials.
    slack = half_step(dtype) * want.abs() + ((half_step(BF16) if dtype == BF16 else 0.0) + 2.0**-15) * size
    if dtype == BF16:
        slack = slack + case.least
    if large:
        # A score is summed in float32: head_dim / 16 steps of the tensor cores, each off by 2^-23 of the sum of magnitudes at
        # most (or head_dim roundings of 2^-24 that go either way): 2^-20 of that sum for 128 dims.  An error e of the scores
        # moves a weight, and the sum that divides it, by a factor of exp(+-e): the output by 2 e of the values' sum.
        slack = slack + 2 * 2.0**-20 * case.reach(q, heads, scale) * size
    bad = ((got - want).abs() > slack + tiny) & fine
    assert not bool(bad.any()), (float(((got - want).abs() / size.clamp(min=1e-30))[bad].max()), bad.nonzero()[:4].tolist())
    return got


HEADS = [  # query heads, kv heads, key size, value size
    (12, 2, 128, 128), (28, 4, 128, 128), (8, 8, 64, 64), (40, 2, 128, 128), (6, 2, 64, 64), (3, 1, 48, 48), (4, 2, 32, 24), (5, 5, 256, 256),
    (2, 1, 128, 64), (1, 1, 16, 16), (32, 1, 64, 64), (3, 3, 33, 7),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [16, 5, 64])
@pytest.mark.parametrize("heads", HEADS)
def test_single_tokens_over_8_bits(sets, dtype, heads, page):
    h, kv, dim, vdim = heads
    check(sets[dtype], Case("single", [(0, 1), (1, 1), (15, 1), (16, 1), (300, 1), (1023, 1), (31, 1)], kv, dim, vdim, page, E4M3, dtype, DEV), h)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("what", [dict(window=1), dict(window=33), dict(chunk=64), dict(window=20, keep_first=4), dict(window=100, keep_first=37),
                                  dict(softcap=5.0), dict(sink=1.5), dict(window=50, softcap=30.0, sink=-2.0, keep_first=3)])
def test_what_single_tokens_see(sets, dtype, what):
    what = dict(what)
    if "sink" in what:
        what["sink"] = what["sink"] + torch.randn(12, generator=torch.Generator().manual_seed(4)).to(DEV)
    check(sets[dtype], Case("single", [(0, 1), (63, 1), (64, 1), (500, 1), (129, 1)], 2, 128, 128, 16, E4M3, dtype, DEV), 12, **what)


@pytest.mark.parametrize("requests,longest", [(1, 9000), (2, 40000), (70, 900)])
def test_long_and_many_single_tokens(sets, requests, longest):
    case = Case("single", [(max(0, longest - 211 * i % longest), 1) for i in range(requests)], 2, 128, 128, 16, E4M3, BF16, DEV)
    check(sets[BF16], case, 14)


def test_a_mixed_step_over_8_bits(sets):
    """Single tokens on the numbers as they are, portions on the pages read back, in one call."""
    for dtype, heads in ((BF16, (12, 2, 128, 128)), (BF16, (4, 2, 48, 48)), (F32, (4, 2, 64, 64)), (BF16, (4, 2, 80, 40))):
        h, kv, dim, vdim = heads
        case = Case("portion", [(100, 1), (7, 1), (50, 3), (0, 200), (301, 130)], kv, dim, vdim, 16, E4M3, dtype, DEV)
        case.masks = [torch.ones(n, n).tril().bool() for n in case.news]
        for what in ({}, dict(window=64), dict(chunk=50), dict(softcap=10.0, sink=torch.randn(h, generator=torch.Generator().manual_seed(1)).to(DEV))):
            # pages read back are rounded to the engine's type once more: half a step of a key moves a score, of a value the sum.
            q = queries(case, h, dtype) / 4
            out = torch.empty((case.step.num_tokens, h * vdim), dtype=dtype, device=DEV)
            sets[dtype].attention(q, out, case.step, case.kv, h, kv, dim, what.get("window"), dim**-0.5, what.get("chunk"), 0,
                                  what.get("softcap", 0.0), what.get("sink"))
            sets[dtype].check_errors()
            want, size = case.attention(q, h, dim**-0.5, **what)
            # |q| |k| of up to 6 a score and a rounded key moves it by at most 2^-8 of that; weights move as much; tanh of 16-bit sets: 2^-11 * 10.
            moved = (6.0 * half_step(BF16) + 3 * half_step(BF16) + 10 * 2.0**-11) if dtype == BF16 else 2.0**-15
            assert bool(((out.double().cpu() - want).abs() <= half_step(dtype) * want.abs() + 2 * moved * size).all())


TREES = [
    [(0, [-1])],
    [(300, [-1, 0, 1, 2, 3])],
    [(0, [-1, 0, 0, -1, 2]), (17, [-1]), (1000, random_parents(64, 1)), (129, random_parents(33, 2))],
    [(2000, random_parents(256, 3)), (5, random_parents(100, 4))],
    [(64, random_parents(7, 5)) for _ in range(40)],
]


@pytest.mark.parametrize("t", range(len(TREES)))
@pytest.mark.parametrize("cache", [E4M3, BF16, F32])
@pytest.mark.parametrize("heads", [(12, 2, 128, 128), (4, 4, 64, 64), (7, 1, 128, 128), (3, 1, 48, 40), (40, 2, 64, 64)])
def test_trees(sets, t, cache, heads):
    h, kv, dim, vdim = heads
    for dtype in ((BF16, F32) if cache == E4M3 else (cache,)):
        check(sets[dtype], Case("tree", TREES[t], kv, dim, vdim, 16, cache, dtype, DEV, seed=t), h)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
@pytest.mark.parametrize("what", [dict(window=1), dict(window=3), dict(window=33), dict(window=700), dict(chunk=64), dict(window=20, keep_first=4),
                                  dict(window=2, keep_first=30), dict(softcap=5.0), dict(sink=1.0), dict(window=50, softcap=30.0, sink=-2.0)])
def test_what_trees_see(sets, dtype, cache, what):
    what = dict(what)
    if "sink" in what:
        what["sink"] = what["sink"] + torch.randn(12, generator=torch.Generator().manual_seed(4)).to(DEV)
    case = Case("tree", [(0, random_parents(9, 1)), (62, random_parents(20, 2)), (900, list(range(-1, 70))), (2, [-1, 0, 1, 2, 3, -1])], 2, 128, 128, 16,
                cache, dtype, DEV)
    check(sets[dtype], case, 12, **what)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32)])
def test_masks_of_any_form_and_rows_that_see_nothing(sets, dtype, cache):
    g = torch.Generator().manual_seed(8)
    masks = [torch.rand(40, 40, generator=g) < 0.3, torch.rand(70, 70, generator=g) < 0.1]
    masks[0][3], masks[0][17], masks[1][:5] = False, False, False
    case = Case("tree", [(0, [-1] * 40), (0, list(range(-1, 69)))], 2, 128, 128, 16, cache, dtype, DEV, masks=masks)
    got = check(sets[dtype], case, 12)
    empty = ~torch.cat([m.any(1) for m in masks])
    assert bool((got[empty] == 0).all()) and int(empty.sum()) >= 7
    check(sets[dtype], case, 12, sink=torch.randn(12, generator=g).to(DEV))


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
@pytest.mark.parametrize("dim", [128, 48])
def test_numbers_that_are_not_finite_reach_those_that_see_them(sets, dtype, cache, dim):
    """In a new token's key or value, in rows of the last page behind the request's end, and behind a window."""
    case = Case("tree", [(200, [-1, 0, 0, 1, 2]), (37, [-1, 0, 1])], 2, dim, dim, 16, cache, dtype, DEV)
    spoiled = float("nan")

    def spoil(which, request, place, value):
        page = int(case.table[case.seats[request], place // 16])
        if cache == E4M3:
            getattr(case.kv, which + "_scale")[page, :, place % 16] = spoiled
            getattr(case.kv, which).view(torch.uint8)[page, :, place % 16] = 0
        else:
            getattr(case.kv, which)[page, :, place % 16, 3] = value

    spoil("v", 0, 200 + 2, spoiled)   # seen by node 2 and its child 4
    spoil("k", 1, 37 + 2, spoiled)    # seen by node 2
    for place in range(40, 48):       # rows of the last page that belong to nobody
        spoil("v", 1, place, float("inf"))
        spoil("k", 1, place, spoiled)
    got = check(sets[dtype], case, 4)
    assert got[:, :].isnan().any(1).tolist() == [False, False, True, False, True, False, False, True]
    spoil("v", 0, 11, float("inf"))   # behind the window
    check(sets[dtype], case, 4, window=150)
    single = Case("single", [(37, 1)], 2, dim, dim, 16, cache, dtype, DEV)
    if cache == E4M3:
        page = int(single.table[single.seats[0], 2])
        single.kv.v_scale[page, :, 6:] = spoiled
        single.kv.k_scale[page, :, 6:] = spoiled
        assert bool(torch.isfinite(check(sets[dtype], single, 4)).all())
        single.kv.v_scale[page, :, 5] = spoiled
        assert bool(check(sets[dtype], single, 4).isnan().all())


def test_scales_of_very_different_size(sets):
    """Rows a million times larger or smaller than others: weights and scales are multiplied without loss of range."""
    for kind, requests in (("single", [(700, 1), (40, 1)]), ("tree", [(700, [-1, 0, 1, 1]), (40, [-1, 0])])):
        for power in (-30.0, 0.0, 30.0):
            case = Case(kind, requests, 2, 128, 128, 16, E4M3, BF16, DEV)
            g = torch.Generator().manual_seed(3)
            case.kv.v_scale *= (2.0 ** (power + 20 * torch.randn(case.kv.v_scale.shape, generator=g).clamp(-1, 1))).to(DEV)
            check(sets[BF16], case, 12)


def test_large_queries_and_strided_rows(sets):
    for kind, requests in (("single", [(90, 1), (401, 1)]), ("tree", [(90, [-1, 0, 0]), (401, [-1, 0])])):
        case = Case(kind, requests, 2, 128, 128, 16, E4M3, BF16, DEV)
        q = queries(case, 12, BF16, pad=64)
        q[:, 128:256] *= 1e4  # a head whose scores leave one key
        check(sets[BF16], case, 12, q=q, large=True)
        small = q.clone()
        small[:, :256] *= 1e-20
        check(sets[BF16], case, 12, q=small)


def test_two_streams_and_captured_calls(sets):
    """Calls on two streams at once, and a captured call replayed on other numbers, leave one another alone."""
    k = sets[BF16]
    cases = [Case("single", [(3000, 1), (77, 1)], 2, 128, 128, 16, E4M3, BF16, DEV, seed=i) for i in range(2)]
    cases += [Case("tree", [(3000, random_parents(9, i)), (77, [-1])], 2, 128, 128, 16, (E4M3, BF16)[i], BF16, DEV, seed=i) for i in range(2)]
    qs = [queries(c, 12, BF16, seed=i) for i, c in enumerate(cases)]
    outs = [torch.empty_like(q) for q in qs]
    call = lambda i: k.attention(qs[i], outs[i], cases[i].step, cases[i].kv, 12, 2, 128, None, 128**-0.5)  # noqa: E731
    for i in range(4):
        call(i)
    alone = [o.clone() for o in outs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(i)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, alone))
    graphs = []
    for i in range(4):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(i)
        graphs.append(graph)
    other = [queries(c, 12, BF16, seed=50 + i) for i, c in enumerate(cases)]
    for i in range(4):
        qs[i].copy_(other[i])
        outs[i].zero_()
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    replayed = [o.clone() for o in outs]
    for i in range(4):
        call(i)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, replayed))
    k.check_errors()


def test_missing_pages_are_reported(sets):
    from distie_b200.kernels.library import KernelError

    for dtype, cache in ((BF16, E4M3), (BF16, BF16), (F32, F32)):
        for dim in (128, 48):
            kinds = (("tree", [(40, [-1, 0]), (9, [-1])], "drafted"),) + ((("single", [(40, 1), (9, 1)], "decoded"),) if cache == E4M3 else ())
            for kind, requests, word in kinds:
                case = Case(kind, requests, 2, dim, dim, 16, cache, dtype, DEV)
                case.kv.block_table[case.seats[0], 1] = -1 if dim == 128 else case.kv.num_pages
                q = queries(case, 4, dtype)
                out = torch.empty_like(q)
                sets[dtype].attention(q, out, case.step, case.kv, 4, 2, dim, None, 0.1)
                with pytest.raises(KernelError, match=word):
                    sets[dtype].check_errors()
