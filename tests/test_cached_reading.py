"""Pages read back: what is launched, in which order, for the layers of a step."""

from __future__ import annotations

import pytest
import torch

from distie_b200.kernels import cached
from test_cached_refusals import PAGES, Checks, slot, step


@pytest.fixture
def launches(monkeypatch):
    made = []
    monkeypatch.setattr(cached, "packed", lambda name: (lambda block: made.append((name, block)) or 0, lambda *args: args))
    return made


@pytest.mark.parametrize("portions", [1, 9, 300])
def test_the_table_of_pages_read_back_is_made_before_the_pages_and_once_a_step(launches, portions):
    """The attention behind the read looks at the table before it waits for anything, so the launch that fills it may not be the
    one that the attention starts beside."""
    s = step(2 * portions, num_seqs=portions, num_decode_tokens=0, portions=[(3, 2)] * portions)
    reads = -(-portions // 256)
    first = Checks().kv_read(s, slot())
    assert [name for name, _ in launches] == ["distie_rows_table"] * reads + ["distie_rows_read"] * reads
    table = first.block_table.data_ptr()
    assert all(block[4] == table for name, block in launches if name == "distie_rows_table")
    assert not any(table in block for name, block in launches if name == "distie_rows_read")
    launches.clear()
    again = Checks().kv_read(s, slot())  # the next layer of the step
    assert [name for name, _ in launches] == ["distie_rows_read"] * reads and again.block_table is first.block_table
    launches.clear()
    Checks().kv_read(s, slot(), window=2)  # a layer that sees other pages has a table of its own
    Checks().kv_read(s, slot(block_table=torch.zeros(2, PAGES + 1, dtype=torch.int32)))
    assert [name for name, _ in launches].count("distie_rows_table") == 2 * reads
