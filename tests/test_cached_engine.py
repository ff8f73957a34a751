"""Caches in eight bits and drafted tokens through the engine: configuration, cache manager, batches, generation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import helpers
import plain_qwen2 as plain
from ref_cached import RefCached
from ref_kernels import RefKernels

from distie_b200.cache import CacheManager, pages_that_fit
from distie_b200.config import EngineConfig, get_architecture
from distie_b200.engine.batch import BatchEntry, StepStaging, lay_out
from distie_b200.engine.engine import Engine
from distie_b200.engine.trace_replay import TraceSession
from distie_b200.kernels.interface import E4M3, MOST_DRAFTED
from distie_b200.parts.base import CacheNeed, StateNeed

GPU = pytest.param("cuda:0", marks=pytest.mark.gpu)


def engine_for(name, device="cpu", dtype="float32", cache_dtype="auto", blocks=96, **knobs):
    cfg, page, weights = helpers.tiny(name)
    arch = get_architecture(cfg["architectures"][0])
    config = EngineConfig(num_blocks=blocks * 16 // page, page_size=page, max_seqs=8, dtype=dtype, device=device, cache_dtype=cache_dtype,
                          **{"token_budget": 4096, "decode_graphs": device != "cpu", **knobs})
    torch_dtype = {"float32": torch.float32, "bfloat16": torch.bfloat16}[dtype]
    if device == "cpu":
        kernels = RefCached(torch_dtype)
    else:
        from distie_b200.kernels import make_kernels

        kernels = make_kernels(torch_dtype, device)
    return Engine.assemble(arch, arch.config_cls.from_dict(cfg), weights, kernels, config), cfg, weights


# -- trees as a batch -------------------------------------------------------------------------------------------
def test_a_tree_is_laid_out_by_depth_and_place():
    entries = [BatchEntry(3, [5, 6, 7, 8], 10, (0, 3), [-1, 0, 0, 2]), BatchEntry(1, [9], 4, (0,)), BatchEntry(2, [1, 2, 3], 0, ())]
    layout = lay_out(entries, 100)
    step, rows = StepStaging(200, torch.device("cpu")).upload(layout)
    assert step.positions.tolist() == [4, 10, 11, 11, 12, 0, 1, 2] and step.slots.tolist() == [4, 10, 11, 12, 13, 0, 1, 2]
    assert step.token_ids.tolist() == [9, 5, 6, 7, 8, 1, 2, 3] and step.seq_seat.tolist() == [1, 3, 2]
    assert step.tree.seqs.tolist() == [[0, 1, 4], [1, 4, 10], [5, 3, 0]] and step.tree.most_nodes == 4
    assert step.tree.bits[:, 0].tolist() == [1, 1, 0b11, 0b101, 0b1101, 1, 0b11, 0b111]
    assert rows.tolist() == [1, 4, 0] and step.num_decode_tokens == 0 and step.q_tiles is None and step.max_kv_len == 14


def test_masks_of_large_trees_fill_their_words():
    n = MOST_DRAFTED
    layout = lay_out([BatchEntry(0, [1] * n, 7, (), list(range(-1, n - 1))), BatchEntry(1, [1], 0, ())])
    step, _ = StepStaging(20 * n, torch.device("cpu")).upload(layout)
    bits = step.tree.bits.numpy().view(np.uint32)
    assert bits.shape == (n + 1, 8)
    for t, node in ((0, 0), (1, 0), (32, 31), (33, 32), (n, n - 1)):
        seen = sum(int(w) << (32 * i) for i, w in enumerate(bits[t]))
        assert seen == (1 << (node + 1)) - 1


@pytest.mark.parametrize("parents,word", [([0, 0], "parent"), ([-1, 1], "parent"), ([-1, -2], "parent"), ([-1], "parents for"), ([-1, 0, 1], "parents for")])
def test_trees_that_are_none_are_refused(parents, word):
    with pytest.raises(ValueError, match=word):
        lay_out([BatchEntry(0, [1, 2], 0, (), parents)])


def test_too_many_drafted_tokens_are_refused():
    n = MOST_DRAFTED + 1
    with pytest.raises(ValueError, match="up to"):
        lay_out([BatchEntry(0, [1] * n, 0, (), list(range(-1, n - 1)))])
    with pytest.raises(ValueError, match="up to"):  # (the entries beside a tree are chains)
        lay_out([BatchEntry(0, [1], 0, (), [-1]), BatchEntry(1, [1] * n, 0, ())])


def test_models_whose_layers_cannot_branch_refuse_trees():
    engine, _, _ = engine_for("A")
    seat = engine.cache.open_seat()
    engine.cache.grow(seat, 4)
    engine.model.blocks[0].mixer.tree_safe = False
    fresh = type(engine.runner)(engine.model, engine.cache, 64, 4, False)
    with pytest.raises(ValueError, match="drafted tokens branch"):
        fresh.step([BatchEntry(seat, [1, 2], 0, (0,), [-1, 0])])
    plain_set = RefKernels(torch.float32)
    engine.model.blocks[0].mixer.tree_safe = True
    engine.model.kernels = plain_set
    fresh = type(engine.runner)(engine.model, engine.cache, 64, 4, False)
    with pytest.raises(ValueError, match="drafted tokens branch"):
        fresh.step([BatchEntry(seat, [1, 2], 0, (0,), [-1, 0])])


# -- the cache manager ----------------------------------------------------------------------------------------------
def test_an_8_bit_cache_is_counted_with_its_scales():
    needs = {0: CacheNeed(2, 16), 1: CacheNeed(2, 16)}
    cache = CacheManager(needs, num_pages=5, page_size=4, max_seats=2, max_tokens_per_request=16, dtype=torch.float32, device="cpu", cache_dtype=E4M3)
    assert cache.bytes_per_token() == 2 * 2 * (32 + 8)
    slot = cache.kv_slot(1)
    assert slot.k.dtype == E4M3 and slot.k.shape == (6, 2, 4, 16) and slot.k_scale.shape == (6, 2, 4) and slot.v_scale.dtype == torch.float32
    assert slot.k_scale.data_ptr() != slot.v_scale.data_ptr() and slot.k_scale.is_contiguous()
    assert pages_that_fit(needs, 4, 1, 160 * 4 * 11, 8) == 10
    plain_cache = CacheManager(needs, num_pages=5, page_size=4, max_seats=2, max_tokens_per_request=16, dtype=torch.float32, device="cpu")
    assert plain_cache.kv_slot(0).k_scale is None and plain_cache.bytes_per_token() == 2 * 2 * 32 * 4


def test_what_an_8_bit_cache_does_not_hold_is_refused():
    latent = {0: CacheNeed(1, 24, value_dim=16, values_in_keys=True)}
    with pytest.raises(ValueError, match="eight bits"):
        CacheManager(latent, num_pages=4, page_size=4, max_seats=2, max_tokens_per_request=16, device="cpu", cache_dtype=E4M3)
    with pytest.raises(ValueError, match="a cache holds"):
        CacheManager({0: CacheNeed(1, 8)}, num_pages=4, page_size=4, max_seats=2, max_tokens_per_request=16, device="cpu", cache_dtype=torch.float16)
    with pytest.raises(ValueError, match="cache_dtype"):
        EngineConfig(cache_dtype="int8")
    cfg, page, weights = helpers.tiny("A")
    arch = get_architecture(cfg["architectures"][0])
    with pytest.raises(ValueError, match="serves no cache"):
        Engine.assemble(arch, arch.config_cls.from_dict(cfg), weights, RefKernels(torch.float32),
                        EngineConfig(num_blocks=8, dtype="float32", device="cpu", cache_dtype="float8_e4m3"))


@pytest.mark.parametrize("cache_dtype", [torch.float32, E4M3])
@pytest.mark.parametrize("device", ["cpu", GPU])
def test_kept_places_move_up(device, cache_dtype):
    needs = {0: CacheNeed(2, 8), 1: CacheNeed(1, 8, value_dim=4), 2: CacheNeed(2, 8)}
    cache = CacheManager(needs, num_pages=12, page_size=4, max_seats=2, max_tokens_per_request=32, dtype=torch.float32, device=device,
                         cache_dtype=cache_dtype)
    other, seat = cache.open_seat(), cache.open_seat()
    assert cache.grow(other, 9) and cache.grow(seat, 17)
    g = torch.Generator().manual_seed(0)
    tensors = []
    for group in cache.groups:
        for t in (group._keys, group._values):
            tensors.append(t.view(torch.uint8) if t.dtype == E4M3 else t)
            tensors[-1].copy_((torch.rand(t.shape, generator=g) * 100).to(tensors[-1].dtype))
        if group._scales is not None:
            group._scales.copy_(torch.rand(group._scales.shape, generator=g))
            tensors.append(group._scales)
    before = [t.clone() for t in tensors]
    tables = [group.host_table[seat].copy() for group in cache.groups]
    assert cache.keep_places(seat, 6, [0, 2, 3, 7, 10]) == 11
    places = {7: 8, 8: 9, 9: 13, 10: 16}  # target: source
    at = 0
    for group, table in zip(cache.groups, tables):
        for t, old in zip(tensors[at : at + (3 if cache_dtype == E4M3 else 2)], before[at:]):
            want = old.clone()
            lead = (slice(None),) * (2 if t is group._scales else 1)
            for to, source in places.items():
                want[(*lead, table[to // 4], slice(None), to % 4)] = old[(*lead, table[source // 4], slice(None), source % 4)]
            assert torch.equal(t, want)
        at += 3 if cache_dtype == E4M3 else 2
    assert cache.keep_places(seat, 6, [0, 1, 2]) == 9 and cache.keep_places(seat, 6, []) == 6  # nothing moves
    for bad in ([1, 1], [2, 1], [-1]):
        with pytest.raises(ValueError, match="rising"):
            cache.keep_places(seat, 6, bad)
    with pytest.raises(ValueError, match="holds no page"):
        cache.keep_places(seat, 6, [0, 20])
    with pytest.raises(ValueError, match="longest"):
        cache.keep_places(seat, 6, [40])
    cache.close_seat(seat)
    with pytest.raises(ValueError, match="not open"):
        cache.keep_places(seat, 0, [0])
    states = CacheManager({}, {0: StateNeed((2,))}, num_pages=1, page_size=4, max_seats=1, max_tokens_per_request=8, device="cpu")
    with pytest.raises(ValueError, match="state"):
        states.keep_places(states.open_seat(), 0, [1])


# -- drafted tokens through the engine ----------------------------------------------------------------------------------
TREE = [-1, 0, 0, 1, 1, 2, 5, -1, 7, 3]


def path_to(node, parents):
    path = []
    while node >= 0:
        path.append(node)
        node = parents[node]
    return path[::-1]


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("name", ["A", "B", "D", "E"])
def test_a_tree_step_gives_the_logits_of_every_path(name, device):
    """Trees of several requests beside a single token, then a kept path, then ordinary steps over the rows it left."""
    engine, cfg, weights = engine_for(name, device)
    vocab = cfg["vocab_size"]
    prompts = [helpers.random_ids(vocab, n, 60 + n) for n in (21, 1, 40)]
    seats = [engine.cache.open_seat() for _ in prompts]
    for seat, ids in zip(seats, prompts):
        assert engine.cache.grow(seat, len(ids) + 40)
        engine.runner.step([BatchEntry(seat, ids, 0, ())])
    drafts = [helpers.random_ids(vocab, len(TREE), 90), helpers.random_ids(vocab, 3, 91), helpers.random_ids(vocab, 1, 92)]
    trees = [TREE, [-1, 0, 0], [-1]]
    entries = [BatchEntry(s, d, len(p), tuple(range(len(d))), t) for s, d, p, t in zip(seats, drafts, prompts, trees)]
    entries[2].parents = None
    logits = engine.runner.step(entries).float().cpu()
    engine.runner.finish_step()
    got, want, at = {}, {}, 0
    for r, (ids, draft, tree) in enumerate(zip(prompts, drafts, trees)):
        for node in range(len(draft)):
            full = ids + [draft[n] for n in path_to(node, tree)]
            got[f"{r}.{node}"], want[f"{r}.{node}"] = logits[at : at + 1], plain.forward_logits(full, weights, cfg)[-1:]
            at += 1
    error, where, _ = helpers.worst_error(got, want)
    assert error <= helpers.FP32_TOL, (where, error)
    kept = path_to(9, TREE)  # 0, 1, 3, 9
    cached = engine.cache.keep_places(seats[0], len(prompts[0]), kept)
    ids, tail = prompts[0] + [drafts[0][n] for n in kept], helpers.random_ids(vocab, 6, 93)
    expected = plain.forward_logits(ids + tail, weights, cfg)[len(ids) :]
    first = engine.runner.step([BatchEntry(seats[0], tail[:4], cached, (0, 1, 2, 3))]).float().cpu().clone()
    rest = [engine.runner.step([BatchEntry(seats[0], [t], cached + 4 + i, (0,))]).float().cpu().clone() for i, t in enumerate(tail[4:])]
    error, where, _ = helpers.worst_error({"tail": torch.cat([first, *rest])}, {"tail": expected})
    assert error <= helpers.FP32_TOL, error


def drafters(prompt, answer, vocab):
    """Guesses that are all right, all wrong, none, and a tree with the right ones among wrong ones."""
    at = lambda ids: len(ids) - len(prompt)  # noqa: E731

    def right(ids):
        tokens = answer[at(ids) : at(ids) + 5]
        return tokens, list(range(-1, len(tokens) - 1))

    def wrong(ids):
        return [(answer[min(at(ids), len(answer) - 1)] + 1) % vocab], [-1]

    def tree(ids):
        a = answer[at(ids) : at(ids) + 3]
        if len(a) < 3:
            return [], []
        other = (a[0] + 3) % vocab
        return [other, a[0], other, a[1], (a[1] + 1) % vocab, a[1], (a[2] + 2) % vocab, a[2]], [-1, -1, 0, 1, 1, 0, 3, 3]

    return {"right": right, "wrong": wrong, "none": lambda ids: ([], []), "tree": tree}


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("which", ["right", "wrong", "none", "tree"])
def test_drafted_generation_is_greedy_generation(name, device, which):
    engine, cfg, weights = engine_for(name, device, token_budget=32)
    prompt = helpers.random_ids(cfg["vocab_size"], 45, 7)  # (longer than a step takes)
    answer = plain.greedy_generate(prompt, weights, cfg, 21)
    made = engine.generate_drafted(prompt, drafters(prompt, answer, cfg["vocab_size"])[which], 20, eos_id=None)
    assert made.token_ids == answer[:20] and made.finish_reason == "length"
    if which == "right":
        assert made.steps <= 4 and made.accepted >= 15
    elif which == "tree":
        assert made.steps < 12 and made.accepted > 8 and made.drafted > 3 * made.steps
    else:
        assert made.accepted == 0 and made.steps == 19
    assert engine.cache.free_pages() == engine.cache.total_pages() and engine.cache.free_seats == 8
    stop = answer[6]
    made = engine.generate_drafted(prompt, drafters(prompt, answer, cfg["vocab_size"])[which], 20, eos_id=stop)
    assert made.token_ids == answer[: answer.index(stop) + 1] and made.finish_reason == "eos"


def test_drafted_generation_refuses_and_cleans_up():
    engine, cfg, _ = engine_for("A")
    with pytest.raises(ValueError, match="non-empty"):
        engine.generate_drafted([], lambda ids: ([], []))
    with pytest.raises(ValueError, match="parents"):
        engine.generate_drafted([1, 2], lambda ids: ([3], []), 4, eos_id=None)
    with pytest.raises(ValueError, match="parent"):
        engine.generate_drafted([1, 2], lambda ids: ([3], [0]), 4, eos_id=None)
    assert engine.cache.free_pages() == engine.cache.total_pages() and engine.cache.free_seats == 8
    made = engine.generate_drafted([1, 2], lambda ids: ([5] * 400, [-1] * 400), 6, eos_id=None)  # more than a step takes
    assert len(made.token_ids) == 6


# -- an 8-bit cache through the engine ------------------------------------------------------------------------------------
def replayed(engine, requests, schedule):
    return helpers.collect(schedule, helpers.run_schedule(TraceSession(engine), schedule))


def near_enough(got, want):
    """Float32 sums in another order move a number by 1e-6 of its row's largest; a number that lies as near to a border of
    e4m3, one in 1e5 of them (steps are a sixteenth to an eighth of a number), then goes the other way: of the 50,000 to 100,000
    numbers that a run stores about one does, and every later token of its request sees it.  An eighth of one of a
    head's 16 to 128 products moves a score by about 1 / 64 and logits by as much of their scale; a few such, 0.05.  The first
    tokens of a request, whose rows are a fiftieth of all, agree as those of a cache in float32 do."""
    for r in want:
        errors = (got[r].float() - want[r]).abs().amax(-1) / plain.logit_scale(want[r])
        assert float(errors[:3].max()) <= helpers.FP32_TOL and float(errors.max()) <= 0.05, (r, errors.tolist())


@pytest.mark.parametrize("name,device", [("A", "cpu"), ("E", "cpu"), pytest.param("A", "cuda:0", marks=pytest.mark.gpu),
                                         pytest.param("D", "cuda:0", marks=pytest.mark.gpu), pytest.param("E", "cuda:0", marks=pytest.mark.gpu)])
def test_an_8_bit_cache_gives_the_same_however_prompts_are_cut(name, device):
    cfg = helpers.tiny(name)[0]
    requests = {f"r{i}": helpers.random_ids(cfg["vocab_size"], n, 10 + i) for i, n in enumerate([20, 37, 33] if device == "cpu" else [40, 67, 33, 90])}
    whole = replayed(engine_for(name, device, cache_dtype="float8_e4m3")[0], requests, helpers.schedule_whole(requests))
    exact = replayed(engine_for(name, device)[0], requests, helpers.schedule_whole(requests))
    assert max(float((whole[r] - exact[r]).abs().max()) for r in requests) > 0, "the cache is not in eight bits"
    for make in (helpers.schedule_tail, helpers.schedule_portions, helpers.schedule_mixed):
        near_enough(replayed(engine_for(name, device, cache_dtype="float8_e4m3")[0], requests, make(requests)), whole)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "C", "D", "E"])
def test_8_bit_engines_agree_with_the_plain_kernel_set(name):
    cfg = helpers.tiny(name)[0]
    requests = {f"r{i}": helpers.random_ids(cfg["vocab_size"], n, 30 + i) for i, n in enumerate([50, 21, 77])}
    steps = helpers.schedule_mixed(requests)
    want = replayed(engine_for(name, cache_dtype="float8_e4m3")[0], requests, steps)
    near_enough(replayed(engine_for(name, "cuda:0", cache_dtype="float8_e4m3")[0], requests, steps), want)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "C", "D"])
def test_8_bit_bfloat16_engines_generate_with_and_without_graphs(name):
    """Captured decode steps over an 8-bit cache give the tokens that eager steps give; bfloat16 and float32 engines agree as
    far as bfloat16 does with a cache of its own type."""
    prompts = [helpers.random_ids(helpers.tiny(name)[0]["vocab_size"], n, 70 + n) for n in (1, 5, 33, 140)]
    eager, _, _ = engine_for(name, "cuda:0", "bfloat16", "float8_e4m3", decode_graphs=False)
    graphs, cfg, weights = engine_for(name, "cuda:0", "bfloat16", "float8_e4m3")
    made = [r.token_ids for r in eager.generate(prompts, max_new_tokens=24, ignore_eos=True)]
    assert [r.token_ids for r in graphs.generate(prompts, max_new_tokens=24, ignore_eos=True)] == made
    assert graphs.runner.graph_replays > 10 and graphs.runner.use_graphs
    assert graphs.cache.free_pages() == graphs.cache.total_pages()
    counts = graphs.model.kernels.kernel_counts
    assert counts.get("rows_write") and counts.get("rows_read")
    assert counts.get("attention_decode_e4m3" if name in "CD" else "attention_rows")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", ["auto", "float8_e4m3"])
@pytest.mark.parametrize("name", ["C", "D"])
def test_drafted_steps_in_bfloat16_agree_with_single_steps(name, cache_dtype):
    """The logits of a chain of drafted tokens are those of the same tokens one by one, within what bfloat16 costs; and a whole
    generation with drafted trees runs over either cache."""
    engine, cfg, weights = engine_for(name, "cuda:0", "bfloat16", cache_dtype)
    ids, draft = helpers.random_ids(cfg["vocab_size"], 150, 3), helpers.random_ids(cfg["vocab_size"], 40, 4)
    seat, other = engine.cache.open_seat(), engine.cache.open_seat()
    for s in (seat, other):
        engine.cache.grow(s, 200)
        engine.runner.step([BatchEntry(s, ids, 0, ())])
    chain = engine.runner.step([BatchEntry(seat, draft, 150, tuple(range(40)), list(range(-1, 39)))]).float().cpu()
    single = torch.cat([engine.runner.step([BatchEntry(other, [t], 150 + i, (0,))]).float().cpu() for i, t in enumerate(draft)])
    engine.runner.finish_step()
    expected = {"r": plain.forward_logits(ids + draft, weights, cfg)[150:]}
    budget = helpers.Bf16Budget({"r": ids + draft}, weights, cfg, expected, skip=150)
    if cache_dtype == "auto":
        budget.check({"r": chain}, expected, "a chain of drafted tokens")
    # Both sides are off by as much as bfloat16 costs, over the same cache: together twice that, 8-bit rounding of rows that went
    # another way left aside (see near_enough).
    worst, rms, _ = helpers.pooled_stats({"r": chain}, {"r": single})
    assert rms <= 2 * budget.rms_error + (0.01 if cache_dtype != "auto" else 0.0), rms
    answer = [r.token_ids for r in engine.generate([ids], max_new_tokens=30, ignore_eos=True)][0]
    made = engine.generate_drafted(ids, drafters(ids, answer, cfg["vocab_size"])["tree"], 24, eos_id=None)
    assert len(made.token_ids) == 24 and made.accepted > 0
    assert engine.model.kernels.kernel_counts.get("attention_tree_tcgen05")


@pytest.mark.gpu
def test_an_8_bit_engine_is_sized_from_free_memory_and_preempts():
    engine, cfg, _ = engine_for("B", "cuda:0", "bfloat16", "float8_e4m3", prefill_chunk=helpers.TINY_B_CHUNK)
    prompts, results = helpers.run_tiny_b_workload(engine, cfg)
    assert all(len(r.token_ids) == helpers.TINY_B_STEPS for r in results) and results[4].preemptions >= 1
    sized, _, _ = engine_for("B", "cuda:0", "bfloat16", "float8_e4m3", gpu_mem_fraction=0.0005)
    plain_sized, _, _ = engine_for("B", "cuda:0", "bfloat16", gpu_mem_fraction=0.0005)
    need = 2 * 32  # elements of a token's key and value: 128 bytes in bfloat16, 64 + 8 in eight bits
    assert sized.cache.total_pages() / plain_sized.cache.total_pages() == pytest.approx(2 * need / (need + 8), rel=0.05)
