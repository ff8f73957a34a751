"""Attention over cached keys whose scores rise, fall and jump: the maximum in use of a softmax is left behind again and again,
inside a block of keys and between blocks, by a few powers of two and by hundreds, against 64 bits."""

from __future__ import annotations

import pytest
import torch

from plain_cached import E4M3, Case
from test_cached_attention_gpu import BF16, DEV, F32, check

pytestmark = pytest.mark.gpu
KEYS = 700


@pytest.fixture(scope="module")
def sets():
    from distie_b200.kernels import make_kernels

    return {dtype: make_kernels(dtype, DEV) for dtype in (BF16, F32)}


def profile(what, n):
    """A score (in nats, of the head that takes it as it is) for each of n keys."""
    j = torch.arange(n, dtype=torch.float64)
    if what.startswith("rise"):  # by so much in 32 keys
        return j * (float(what[4:]) / 32)
    if what.startswith("fall"):
        return (n - j) * (float(what[4:]) / 32)
    s = torch.zeros(n, dtype=torch.float64)
    if what == "jumps":  # at the first, last and neighbouring keys of groups, halves and blocks
        for height, at in enumerate((0, 31, 32, 33, 63, 64, 95, 96, 127, 128, 159, 300, 511, 512, n - 1)):
            s[at:] = 12.0 * height
        return s
    if what == "spikes":
        for height, at in enumerate((5, 40, 41, 70, 100, 129, 200, 255, 256, 400, n - 2)):
            s[at % n] = 9.0 * (height + 1)
        return s
    assert what == "waves"
    return 25.0 * torch.sin(j / 11) + j / 16


def shaped(kind, cache, dtype, dim, what):
    requests = [(KEYS, 1), (333, 1)] if kind == "single" else [(KEYS, [-1, 0, 0, 1, 3]), (333, [-1, -1, 1])]
    case = Case(kind, requests, 2, dim, dim, 16, cache, dtype, DEV)
    g = torch.Generator().manual_seed(5)
    u = torch.randn(dim, generator=g, dtype=torch.float64).to(E4M3).double()
    unit = u / (u @ u)
    for r, (past, new) in enumerate(zip(case.pasts, case.news)):
        s = profile(what, past + new)
        pages = case.table[case.seats[r], torch.arange(past + new) // case.page].long().to(DEV)
        rows = (torch.arange(past + new) % case.page).to(DEV)
        for kv in range(2):
            if cache == E4M3:  # the row u, or its opposite, times a scale
                numbers = torch.where(s[:, None] >= 0, u[None], -u[None]).to(E4M3).to(DEV)
                case.kv.k.view(torch.uint8)[pages, kv, rows] = numbers.view(torch.uint8)
                case.kv.k_scale[pages, kv, rows] = (s.abs() + 1e-3).float().to(DEV)
            else:
                case.kv.k[pages, kv, rows] = (s[:, None] * u[None]).to(dtype).to(DEV)
    heads = 12
    turn = torch.tensor([1.0, -1.0, 0.5, 0.01, -0.1, 2.0], dtype=torch.float64).repeat(2)  # heads see the profile turned over, flatter, steeper
    q = (turn[:, None] * unit * dim**0.5).reshape(1, -1).expand(case.step.num_tokens, -1)
    return case, q.to(dtype).contiguous().to(DEV), heads


def lost(case):
    """Weights below 2^-126 of the largest (or of the sink's) are zeros: float32 exponentials end there.  An output misses at most
    that much of every key's value."""
    return 2.0**-126 * KEYS * float(case.rows("v").abs().amax())


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("what", ["rise3", "rise12", "rise60", "rise700", "fall12", "fall700", "jumps", "spikes", "waves"])
@pytest.mark.parametrize("kind, cache, dtype, dim", [
    ("single", E4M3, BF16, 128), ("single", E4M3, BF16, 64), ("tree", E4M3, BF16, 128), ("tree", E4M3, BF16, 64), ("tree", BF16, BF16, 128),
    ("tree", BF16, BF16, 64), ("tree", E4M3, F32, 64), ("tree", F32, F32, 48),
])
def test_maxima_left_behind(sets, monkeypatch, kind, cache, dtype, dim, what, splits):
    from distie_b200.kernels import cached

    monkeypatch.setattr(cached, "tree_splits", lambda *_: splits)
    monkeypatch.setattr(cached, "decode_splits", lambda *_: splits)
    case, q, heads = shaped(kind, cache, dtype, dim, what)
    check(sets[dtype], case, heads, q=q, large=True)
    check(sets[dtype], case, heads, q=q, large=True, window=200, keep_first=33)
    check(sets[dtype], case, heads, q=q, large=True, tiny=lost(case), sink=torch.linspace(-20.0, 60.0, heads, device=DEV))


@pytest.mark.parametrize("kind", ["single", "tree"])
def test_values_whose_scales_rise_against_the_scores(sets, monkeypatch, kind):
    """Weights times scales have a maximum of their own: here far from the softmax's, and moving the other way."""
    from distie_b200.kernels import cached

    monkeypatch.setattr(cached, "tree_splits", lambda *_: 1)
    monkeypatch.setattr(cached, "decode_splits", lambda *_: 1)
    for what, turn in (("fall12", 1.0), ("rise12", -1.0), ("rise3", 2.0), ("spikes", 3.0)):
        case, q, heads = shaped(kind, E4M3, BF16, 128, what)
        for r, (past, new) in enumerate(zip(case.pasts, case.news)):
            pages = case.table[case.seats[r], torch.arange(past + new) // case.page].long().to(DEV)
            rows = (torch.arange(past + new) % case.page).to(DEV)
            case.kv.v_scale[pages, :, rows] *= torch.exp(turn * torch.arange(past + new) / 20.0).clamp(1e-25, 1e25).float().to(DEV)[:, None]
        check(sets[BF16], case, heads, q=q, large=True)
