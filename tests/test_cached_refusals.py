"""What the kernels of 8-bit caches and drafted tokens refuse, before anything is launched."""

from __future__ import annotations

import contextlib

import pytest
import torch

from distie_b200.kernels import DraftTree, cached
from distie_b200.kernels.cached import CachedRows, decode_splits, rows_splits, tree_splits
from distie_b200.kernels.interface import E4M3, KvSlot, RotaryTable, StepTensors
from distie_b200.kernels.library import KernelError

HEADS, KV, DIM, PAGE, PAGES = 6, 2, 32, 8, 4


class Checks(CachedRows):
    """The checks of the CUDA sets, on the host."""

    dtype, sm_count = torch.bfloat16, 148

    def __init__(self):
        self.error_flag = torch.zeros(1, dtype=torch.int32)

    def _here(self):
        return contextlib.nullcontext()

    def _stream(self):
        return 0

    def _ran(self, name, count=1):
        pass


@pytest.fixture
def checks(monkeypatch):
    def launched(name):
        raise AssertionError(f"{name} would have been launched")

    monkeypatch.setattr(cached, "packed", launched)
    return Checks()


def slot(dtype=E4M3, **other) -> KvSlot:
    shape = (PAGES, KV, PAGE)
    made = dict(k=torch.zeros(*shape, DIM).to(dtype), v=torch.zeros(*shape, DIM).to(dtype), block_table=torch.zeros(2, PAGES, dtype=torch.int32),
                page_size=PAGE, num_pages=PAGES, k_scale=torch.ones(shape) if dtype == E4M3 else None,
                v_scale=torch.ones(shape) if dtype == E4M3 else None)
    return KvSlot(**{**made, **other})


def step(tokens=3, **other) -> StepTensors:
    i32 = dict(dtype=torch.int32)
    made = dict(token_ids=torch.zeros(tokens, **i32), positions=torch.arange(tokens, **i32), token_seq=torch.arange(tokens, **i32),
                seq_seat=torch.zeros(tokens, **i32), num_tokens=tokens, num_seqs=tokens, num_decode_tokens=tokens, max_kv_len=24)
    return StepTensors(**{**made, **other})


def tree(tokens=3, **other) -> DraftTree:
    made = dict(bits=torch.ones(tokens, 1, dtype=torch.int32), seqs=torch.tensor([[0, tokens, 4]], dtype=torch.int32), most_nodes=tokens)
    return DraftTree(**{**made, **other})


def attend(checks, kv=None, s=None, q=None, out=None):
    s = s or step()
    q = torch.zeros(3, HEADS * DIM, dtype=torch.bfloat16) if q is None else q
    out = torch.zeros(3, HEADS * DIM, dtype=torch.bfloat16) if out is None else out
    checks._attention_rows(q, out, s, kv or slot(), HEADS, KV, DIM, 0, 0, DIM**-0.5, 0, 0.0, None, s.num_tokens, s.num_seqs)


def test_a_call_that_fits_is_launched(checks):
    with pytest.raises(AssertionError, match="attention_rows would"):
        attend(checks)
    with pytest.raises(AssertionError, match="attention_rows would"):
        attend(checks, s=step(num_seqs=1, num_decode_tokens=0, tree=tree()))


def test_a_step_without_tokens_launches_nothing(checks):
    s = step(0)
    attend(checks, s=s, q=torch.zeros(0, HEADS * DIM, dtype=torch.bfloat16), out=torch.zeros(0, HEADS * DIM, dtype=torch.bfloat16))


@pytest.mark.parametrize("what, word", [
    (dict(k=torch.zeros(PAGES, KV, PAGE, DIM)), "a cache of"),
    (dict(k=torch.zeros(PAGES, KV, PAGE, DIM), v=torch.zeros(PAGES, KV, PAGE, DIM), k_scale=None, v_scale=None), "a cache of"),
    (dict(num_pages=PAGES + 1), "are expected"),
    (dict(page_size=PAGE * 2), "are expected"),
    (dict(v=torch.zeros(PAGES, KV, PAGE, DIM + 8).to(E4M3)), "are expected"),
    (dict(k=torch.zeros(PAGES, KV, DIM, PAGE).to(E4M3).transpose(2, 3)), "contiguous pages"),
    (dict(block_table=torch.zeros(2, PAGES, dtype=torch.int64)), "int32 block table"),
    (dict(block_table=torch.zeros(2, 2 * PAGES, dtype=torch.int32)[:, ::2]), "contiguous int32 block table"),
    (dict(k_scale=None), "comes with the scales"),
    (dict(v_scale=None), "comes with the scales"),
    (dict(k=torch.zeros(PAGES, KV, PAGE, DIM, dtype=torch.bfloat16), v=torch.zeros(PAGES, KV, PAGE, DIM, dtype=torch.bfloat16)), "and only such"),
    (dict(k_scale=torch.ones(PAGES, KV, PAGE, dtype=torch.bfloat16)), "float32 scales"),
    (dict(v_scale=torch.ones(PAGES, KV, PAGE, 1)), "float32 scales"),
    (dict(v_scale=torch.ones(PAGES, KV, 2 * PAGE)[:, :, ::2]), "float32 scales"),
    (dict(k=torch.empty(PAGES, KV, PAGE, DIM, dtype=E4M3, device="meta")), "a cache on"),
    (dict(v_scale=torch.empty(PAGES, KV, PAGE, device="meta")), "float32 scales"),
])
def test_slots_that_do_not_fit(checks, what, word):
    s = step(portions=[], num_decode_tokens=3)
    with pytest.raises(KernelError, match=word):
        attend(checks, slot(**what))
    with pytest.raises(KernelError, match=word + "|keys of one float type|engine's type"):
        rows = torch.zeros(3, KV * DIM, dtype=torch.bfloat16)
        checks._write_keys("kv_write", rows, rows, s, slot(**what))
    if "v" not in what or "k" in what:  # (a slot may hold values of another size: the heads here do not)
        with pytest.raises(KernelError, match=word + "|engine's type"):
            checks.kv_read(s, slot(**what))


@pytest.mark.parametrize("what", [
    dict(most_nodes=0), dict(most_nodes=257), dict(most_nodes=33), dict(bits=torch.ones(3, 1, dtype=torch.int64)),
    dict(bits=torch.ones(2, 1, dtype=torch.int32)), dict(bits=torch.ones(3, 9, dtype=torch.int32)),
    dict(bits=torch.ones(3, 2, dtype=torch.int32)[:, :1]), dict(seqs=torch.zeros(2, 3, dtype=torch.int32)),
    dict(seqs=torch.zeros(1, 3, dtype=torch.int64)), dict(bits=torch.empty(3, 1, dtype=torch.int32, device="meta")),
])
def test_trees_that_do_not_fit(checks, what):
    with pytest.raises(KernelError, match="a tree of 1 to 256"):
        attend(checks, s=step(num_seqs=1, num_decode_tokens=0, tree=tree(**what)))


@pytest.mark.parametrize("what", [
    dict(q=torch.zeros(3, HEADS * DIM)), dict(out=torch.zeros(3, HEADS * DIM)), dict(q=torch.zeros(2, HEADS * DIM, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, HEADS * DIM - 8, dtype=torch.bfloat16)), dict(out=torch.zeros(3, HEADS * DIM - 8, dtype=torch.bfloat16)),
    dict(q=torch.zeros(HEADS * DIM, 3, dtype=torch.bfloat16).t()),
])
def test_queries_and_outputs_that_do_not_fit(checks, what):
    with pytest.raises(KernelError, match="queries and output"):
        attend(checks, **what)


def project(checks, qkv=None, s=None, kv=None, rotary=None, bias=None, q_out=None, norm=(0, 0.0, None, None)):
    qkv = torch.zeros(3, (HEADS + 2 * KV) * DIM) if qkv is None else qkv
    q_out = torch.zeros(3, HEADS * DIM, dtype=torch.bfloat16) if q_out is None else q_out
    checks._write_projection("qkv_norm_write", qkv, bias, s or step(), kv or slot(), rotary, HEADS, KV, DIM, DIM, q_out, norm)


def table(dim, dtype=torch.float32, numbers=None):
    return RotaryTable(inv_freq=torch.ones(numbers or dim // 2, dtype=dtype), rotary_dim=dim, interleaved=False, factor=1.0)


def test_a_projection_that_fits_is_launched(checks):
    with pytest.raises(AssertionError, match="rows_write would"):
        project(checks, rotary=table(DIM), bias=torch.zeros((HEADS + 2 * KV) * DIM))


@pytest.mark.parametrize("what, word", [
    (dict(qkv=torch.zeros(2, (HEADS + 2 * KV) * DIM)), "a projection"),
    (dict(qkv=torch.zeros(3, (HEADS + 2 * KV) * DIM - 1)), "a projection"),
    (dict(qkv=torch.zeros(3, (HEADS + 2 * KV) * DIM, dtype=torch.float16)), "a projection"),
    (dict(qkv=torch.zeros(2, 3, (HEADS + 2 * KV) * DIM, dtype=torch.bfloat16)), "a projection"),
    (dict(qkv=torch.zeros((HEADS + 2 * KV) * DIM, 3).t()), "a projection"),
    (dict(bias=torch.zeros(DIM)), "float32 bias"),
    (dict(bias=torch.zeros((HEADS + 2 * KV) * DIM, dtype=torch.bfloat16)), "float32 bias"),
    (dict(q_out=torch.zeros(3, HEADS * DIM)), "q goes to"),
    (dict(q_out=torch.zeros(3, HEADS * DIM - 2, dtype=torch.bfloat16)), "q goes to"),
    (dict(q_out=torch.zeros(2, HEADS * DIM, dtype=torch.bfloat16)), "q goes to"),
    (dict(rotary=table(2 * DIM)), "rotary table"),
    (dict(rotary=table(DIM, torch.float64)), "rotary table"),
    (dict(rotary=table(DIM, numbers=2)), "rotary table"),
    (dict(norm=(1, 1e-6, torch.ones(DIM, dtype=torch.bfloat16), None)), "float32 weights"),
    (dict(norm=(1, 1e-6, None, torch.ones(DIM + 1))), "float32 weights"),
    (dict(s=step(slots=torch.zeros(3, dtype=torch.int64))), "place in the cache"),
    (dict(s=step(slots=torch.zeros(2, dtype=torch.int32))), "place in the cache"),
])
def test_projections_that_do_not_fit(checks, what, word):
    with pytest.raises(KernelError, match=word):
        project(checks, **what)


def test_keys_and_values_that_do_not_fit(checks):
    good = torch.zeros(3, KV * DIM, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="rows_write would"):
        checks._write_keys("kv_write", good, good, step(), slot())
    for bad in (good.float(), good[:2], good[:, 1:], torch.zeros(KV * DIM, 3, dtype=torch.bfloat16).t(), good.to(torch.float16)):
        with pytest.raises(KernelError, match="of one float type"):
            checks._write_keys("kv_write", good, bad, step(), slot())


def test_reading_back_wants_an_8_bit_cache_and_the_portions(checks):
    with pytest.raises(KernelError, match="engine's type already"):
        checks.kv_read(step(), slot(torch.bfloat16))
    with pytest.raises(KernelError, match="portions"):
        checks.kv_read(step(num_seqs=4), slot())
    with pytest.raises(KernelError, match="portions"):
        checks.kv_read(step(num_seqs=4, portions=[(0, 1), (0, 1)]), slot())
    assert checks.kv_read(step(portions=[]), slot()).num_pages == 0  # (nothing to read, nothing launched)


def test_shares_of_the_keys():
    """Every rule gives at least one share, at most one for 256 keys (a block of 128 with trees) and never more than 64."""
    for blocks in (1, 2, 8, 32, 147, 148, 149, 256, 444, 445, 5000):
        for keys in (0, 1, 255, 256, 511, 512, 1024, 4099, 30011, 1 << 20):
            for wide in (False, True):
                for many in (False, True):
                    assert 1 <= decode_splits(blocks, keys, 148, wide, many) <= max(1, min(64, keys // 256))
            assert 1 <= rows_splits(blocks, keys, 148) <= max(1, min(64, keys // 64))
            assert 1 <= tree_splits(blocks, -(-keys // 128), 148) <= max(1, min(64, -(-keys // 128)))


def test_drafted_generation_is_refused_before_the_prompt_runs():
    from test_cached_engine import engine_for

    engine, _, _ = engine_for("A")
    engine.runner._takes_trees = False

    def step(entries):
        raise AssertionError("a step has run")

    engine.runner.step = step
    with pytest.raises(ValueError, match="drafted tokens branch"):
        engine.generate_drafted([1, 2, 3], lambda ids: ([], []))
