"""The cache manager: pages of keys and values, block tables, seats, state slots.

Control plane and data plane are separate, as in the reference (worker/src/
inference/kv_cache.py:1-10): a native pool hands out page ids only; the keys and
values live in one device slab per group, indexed by those ids.

* A **group** is a set of cache slots (layers) with the same need: kv heads, head
  size, and either all keys or a window of them.  Each group has its own pool,
  slab and block tables, so a windowed group can give pages back while a full
  group keeps them.
* A **seat** is what a live request holds: row ``seat`` of every group's block
  table and slot ``seat`` of every per-request state tensor.  ``close_seat``
  returns the pages of all groups and the seat.
* ``grow(seat, n)`` makes sure the pages for positions ``< n`` exist in every
  group, all or nothing.  ``trim(seat, n)`` returns the pages of windowed groups
  that no position ``>= n`` can see any more.
* Slab layout per group: ``[slot, 2 (k|v), page, kv_head, page_size, head_dim]``
  with one spare page past the pool's range (id ``num_pages``) that padded rows of
  a captured decode step write to (the reference's spare page,
  worker/src/inference/torch_engine.py:439-446).  Row ``max_seats`` of each table
  is the padding seat: all its entries name the spare page.
* State slots: one tensor ``[max_seats + 1, *shape]`` per slot that declares a
  :class:`~distie_b200.parts.base.StateNeed` (a dict of tensors for a slot that declares
  several by name), zeroed when a seat is opened and when a request is sent back to be
  recomputed.  Layers with a recurrence keep their matrix state and the last inputs of
  their short convolutions here.
* A windowed group whose need names ``keep_first`` keeps the pages that hold the request's first
  that-many positions for as long as the request lives: ``trim`` gives back only the pages between them
  and the window.
* A group whose need names a ``chunk`` gives pages back like a windowed one: no later
  position reads a key from before the chunk the request is in.  A group whose values
  have another size than its keys keeps two slabs instead of one; a group whose values lie
  inside its keys (``values_in_keys``: the latent rows of an attention through a latent) keeps
  keys only, and ``KvSlot.v`` is a view of their first columns.

* A cache in eight bits (``cache_dtype=torch.float8_e4m3fn``) holds e4m3 numbers in its slabs and beside
  them, per row of a token and kv head, a float32 scale: ``[slot, 2 (k|v), page, kv_head, page_size]``.
* ``keep_places`` makes the rows of some of a request's newest places its next ones: what is left of a
  tree of drafted tokens once a path of it has been accepted.

With ``device=None`` the manager keeps only the bookkeeping (no slabs), which is
what the scheduler tests and sizing estimates use.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Mapping

import numpy as np
import torch

from ..kernels.interface import E4M3, KvSlot
from ..parts.base import CacheNeed, StateNeed


class CacheExhausted(RuntimeError):
    """No free seat, or a request that can never fit the pool."""


def pages_needed(tokens: int, page_size: int) -> int:
    if page_size < 1:
        raise ValueError("page_size must be >= 1")
    return 0 if tokens <= 0 else (tokens + page_size - 1) // page_size


SCALE_BYTES = 8  # of a token and kv head in a cache in eight bits: a float32 for its key and one for its value


def pages_that_fit(cache_needs, page_size: int, element_size: int, budget_bytes: int, row_bytes: int = 0) -> int:
    """How many pages per group ``budget_bytes`` of device memory hold (the spare page of every slab included
    in the budget, not in the count): every cache slot keeps keys and values of its own for each page id, and
    ``row_bytes`` more for each token and kv head."""
    per_page = sum(need.num_kv_heads * (need.row_elements * element_size + row_bytes) * page_size for need in cache_needs.values())
    if per_page <= 0:
        raise ValueError("the model declares no cache to size")
    return int(budget_bytes // per_page) - 1


@dataclass
class _SeatPages:
    first: int = 0   # logical index of the first page still held
    ids: list | None = None  # page ids of logical pages first, first + 1, ...
    kept: list | None = None  # page ids of logical pages 0, 1, ... that are held for good, once pages behind them went back

    def __post_init__(self) -> None:
        if self.ids is None:
            self.ids = []
        if self.kept is None:
            self.kept = []


class KvGroup:
    def __init__(self, need: CacheNeed, slots: tuple[int, ...], num_pages: int, page_size: int, max_seats: int,
                 table_width: int, pool) -> None:
        self.need = need
        self.slots = slots
        self.num_pages = num_pages
        self.page_size = page_size
        self.table_width = table_width
        self.pool = pool
        self.seats: dict[int, _SeatPages] = {}
        self.host_table = np.full((max_seats + 1, table_width), -1, dtype=np.int32)
        self.host_table[max_seats, :] = num_pages  # padding seat -> spare page
        self.dirty: dict[int, int] = {}  # seat -> first column that changed since the last upload
        self.slab: torch.Tensor | None = None
        self.device_table: torch.Tensor | None = None
        self._host_tensor: torch.Tensor | None = None
        self._views: dict[int, KvSlot] = {}
        self._uploaded = None  # CUDA event after the last upload: the pinned table waits for it before it changes

    def bytes_per_token(self, element_size: int, row_bytes: int = 0) -> int:
        return len(self.slots) * self.need.num_kv_heads * (self.need.row_elements * element_size + row_bytes)

    # -- bookkeeping --------------------------------------------------------
    def first_needed_page(self, cached: int) -> int:
        """Logical index of the first page a position >= cached can still see."""
        first_key = 0
        if self.need.window is not None:
            first_key = max(first_key, cached - int(self.need.window) + 1)
        if self.need.chunk is not None:
            first_key = max(first_key, cached // int(self.need.chunk) * int(self.need.chunk))
        return first_key // self.page_size

    def missing(self, seat: int | None, tokens: int) -> int:
        held = self.seats.get(seat) if seat is not None else None
        end = pages_needed(tokens, self.page_size)
        if held is None:
            return end
        return max(0, end - (held.first + len(held.ids)))

    def _mark(self, seat: int, column: int) -> None:
        self.dirty[seat] = min(self.dirty.get(seat, column), column)

    def _before_write(self) -> None:
        if self._uploaded is not None:
            self._uploaded.synchronize()

    def grow(self, seat: int, tokens: int) -> None:
        held = self.seats.setdefault(seat, _SeatPages())
        count = self.missing(seat, tokens)
        if count == 0:
            return
        start = held.first + len(held.ids)
        if start + count > self.table_width:
            raise CacheExhausted(
                f"{tokens} tokens need {start + count} pages per request, block tables hold {self.table_width}"
            )
        ids = list(self.pool.allocate(count))
        held.ids.extend(ids)
        self._before_write()
        self.host_table[seat, start : start + count] = ids
        self._mark(seat, start)

    def trim(self, seat: int, cached: int) -> int:
        held = self.seats.get(seat)
        if held is None or (self.need.window is None and self.need.chunk is None):
            return 0
        keep_from = min(self.first_needed_page(cached), held.first + len(held.ids))
        head = pages_needed(int(self.need.keep_first), self.page_size) if self.need.window is not None else 0
        if head and held.first == 0 and not held.kept:
            if keep_from <= head:
                return 0  # nothing lies between the pages kept for good and the window yet
            held.kept, held.ids, held.first = held.ids[:head], held.ids[head:], head
        drop = keep_from - held.first
        if drop <= 0:
            return 0
        self.pool.free(held.ids[:drop])
        self._before_write()
        self.host_table[seat, held.first : keep_from] = -1
        self._mark(seat, held.first)
        del held.ids[:drop]
        held.first = keep_from
        return drop

    def release(self, seat: int) -> None:
        held = self.seats.pop(seat, None)
        if held is None:
            return
        if held.ids or held.kept:
            self.pool.free(held.kept + held.ids)
        self._before_write()
        self.host_table[seat, :] = -1
        self._mark(seat, 0)

    def pages_of(self, seat: int) -> list[int]:
        held = self.seats.get(seat)
        return held.kept + held.ids if held else []

    # -- device side --------------------------------------------------------
    def allocate_device(self, dtype: torch.dtype, device: torch.device) -> None:
        rows = (self.num_pages + 1, self.need.num_kv_heads, self.page_size)
        self._scales = None
        if dtype == E4M3:
            if self.need.values_in_keys:
                raise ValueError("a cache in eight bits holds keys and values of their own: rows that are both (attention through a latent) "
                                 "stay in the engine's type")
            self._scales = torch.zeros((len(self.slots), 2, *rows), dtype=torch.float32, device=device)
        if self.need.values_in_keys:  # one row per token; a value is the head of its key's row
            self._keys = torch.zeros((len(self.slots), *rows, self.need.head_dim), dtype=dtype, device=device)
            self._values = self._keys[..., : self.need.v_dim]
        elif self.need.v_dim == self.need.head_dim:
            self.slab = torch.zeros((len(self.slots), 2, *rows, self.need.head_dim), dtype=dtype, device=device)
            self._keys, self._values = self.slab[:, 0], self.slab[:, 1]
        else:  # values of another size than keys: a slab each
            self._keys = torch.zeros((len(self.slots), *rows, self.need.head_dim), dtype=dtype, device=device)
            self._values = torch.zeros((len(self.slots), *rows, self.need.v_dim), dtype=dtype, device=device)
        self._host_tensor = torch.from_numpy(self.host_table)
        if device.type == "cuda":
            self._host_tensor = self._host_tensor.pin_memory()
            self.host_table = self._host_tensor.numpy()  # keep writing into the pinned copy
        self.device_table = self._host_tensor.to(device, non_blocking=False).clone()
        self.dirty.clear()

    def upload(self, seats) -> None:
        if self.device_table is None:
            return
        copied = False
        for seat in seats:
            column = self.dirty.pop(seat, None)
            if column is None:
                continue
            self.device_table[seat, column:].copy_(self._host_tensor[seat, column:], non_blocking=True)
            copied = True
        if copied and self.device_table.is_cuda:
            if self._uploaded is None:
                self._uploaded = torch.cuda.Event()
            self._uploaded.record()

    def rows_at(self, seat: int, places: list[int]) -> np.ndarray:
        """[page, row in it] of the places of a seat, all of which it has to hold."""
        place = np.asarray(places, dtype=np.int64)
        pages = self.host_table[seat, place // self.page_size].astype(np.int64)
        if bool((pages < 0).any()):
            raise ValueError(f"seat {seat} holds no page for some of the places {places}")
        return np.stack([pages, place % self.page_size])

    def move_rows(self, sources: np.ndarray, targets: np.ndarray) -> None:
        """The rows ``sources`` (of :meth:`rows_at`), in every slot, to ``targets`` (all are read before any is written)."""
        if self.device_table is None:
            return
        index = torch.from_numpy(np.stack([sources, targets])).to(self.device_table.device)
        (from_page, from_row), (to_page, to_row) = index[0], index[1]
        held = [self._keys] if self.need.values_in_keys else [self._keys, self._values]
        held = [t.view(torch.uint8) if t.dtype == E4M3 else t for t in held]  # (numbers of eight bits move as bytes)
        if self._scales is not None:
            held += [self._scales[:, 0], self._scales[:, 1]]
        for rows in held:
            rows[:, to_page, :, to_row] = rows[:, from_page, :, from_row]

    def slot_view(self, slot: int) -> KvSlot:
        view = self._views.get(slot)
        if view is None:
            index = self.slots.index(slot)
            scales = (None, None) if self._scales is None else (self._scales[index, 0], self._scales[index, 1])
            view = KvSlot(self._keys[index], self._values[index], self.device_table, self.page_size, self.num_pages + 1, *scales)
            self._views[slot] = view
        return view


class CacheManager:
    def __init__(
        self,
        cache_needs: Mapping[int, CacheNeed],
        state_needs: Mapping[int, StateNeed] | None = None,
        *,
        num_pages: int,
        page_size: int,
        max_seats: int,
        max_tokens_per_request: int,
        dtype: torch.dtype = torch.bfloat16,
        device=None,
        cache_dtype: torch.dtype | None = None,  # None: ``dtype``; torch.float8_e4m3fn: eight bits and a scale per row
        pool_factory: Callable[[int], object] | None = None,
    ) -> None:
        if num_pages < 1 or page_size < 1 or max_seats < 1 or max_tokens_per_request < 1:
            raise ValueError("num_pages, page_size, max_seats and max_tokens_per_request must be >= 1")
        if pool_factory is None:
            from .block_pool import BlockPool as pool_factory
        self.page_size = page_size
        self.max_seats = max_seats
        self.pad_seat = max_seats
        self.max_tokens_per_request = max_tokens_per_request
        self.dtype = dtype
        self.cache_dtype = cache_dtype if cache_dtype is not None else dtype
        if self.cache_dtype not in (dtype, E4M3):
            raise ValueError(f"a cache holds {dtype} or {E4M3}, not {cache_dtype}")
        self.device = torch.device(device) if device is not None else None
        width = pages_needed(max_tokens_per_request, page_size)
        by_need: dict[CacheNeed, list[int]] = {}
        for slot in sorted(cache_needs):
            by_need.setdefault(cache_needs[slot], []).append(slot)
        self.groups = [
            KvGroup(need, tuple(slots), num_pages, page_size, max_seats, width, pool_factory(num_pages))
            for need, slots in by_need.items()
        ]
        self._group_of = {slot: group for group in self.groups for slot in group.slots}
        self.state_needs = dict(state_needs or {})
        self.states: dict[int, torch.Tensor | dict[str, torch.Tensor]] = {}
        self._free_seats = list(range(max_seats - 1, -1, -1))
        self._open: set[int] = set()
        if self.device is not None:
            for group in self.groups:
                group.allocate_device(self.cache_dtype, self.device)
            def make(need: StateNeed) -> torch.Tensor:
                return torch.zeros((max_seats + 1, *need.shape), dtype=need.dtype, device=self.device)

            for slot, need in self.state_needs.items():
                self.states[slot] = make(need) if isinstance(need, StateNeed) else {n: make(item) for n, item in need.items()}

    # -- seats --------------------------------------------------------------
    @property
    def free_seats(self) -> int:
        return len(self._free_seats)

    def open_seat(self) -> int:
        if not self._free_seats:
            raise CacheExhausted(f"all {self.max_seats} seats are taken")
        seat = self._free_seats.pop()
        self._open.add(seat)
        self._clear_state(seat)
        return seat

    def state_tensors(self) -> list[torch.Tensor]:
        """Every per-request state tensor, ``[max_seats + 1, ...]`` each, in a fixed order."""
        out = []
        for slot in sorted(self.states):
            held = self.states[slot]
            out += [held] if isinstance(held, torch.Tensor) else [held[name] for name in sorted(held)]
        return out

    def _clear_state(self, seat: int) -> None:
        for state in self.state_tensors():
            state[seat].zero_()

    def state_bytes_per_seat(self) -> int:
        return sum(t[0].numel() * t.element_size() for t in self.state_tensors())

    def close_seat(self, seat: int) -> None:
        if seat not in self._open:
            raise ValueError(f"seat {seat} is not open")
        for group in self.groups:
            group.release(seat)
        self._open.remove(seat)
        self._free_seats.append(seat)

    def reset_seat(self, seat: int) -> None:
        """Give back the pages and clear the state but keep the seat (recompute from position 0)."""
        if seat not in self._open:
            raise ValueError(f"seat {seat} is not open")
        for group in self.groups:
            group.release(seat)
        self._clear_state(seat)

    # -- pages --------------------------------------------------------------
    def fits_ever(self, tokens: int) -> bool:
        if tokens > self.max_tokens_per_request:
            return False
        return all(pages_needed(tokens, g.page_size) <= g.num_pages for g in self.groups)

    def can_grow(self, seat: int | None, tokens: int) -> bool:
        return all(g.missing(seat, tokens) <= g.pool.num_free for g in self.groups)

    def grow(self, seat: int, tokens: int) -> bool:
        """Pages for positions < tokens in every group, all or nothing."""
        if seat not in self._open:
            raise ValueError(f"seat {seat} is not open")
        if tokens > self.max_tokens_per_request:
            raise CacheExhausted(f"{tokens} tokens exceed the longest request the tables hold ({self.max_tokens_per_request})")
        if not self.can_grow(seat, tokens):
            return False
        for group in self.groups:
            group.grow(seat, tokens)
        return True

    def trim(self, seat: int, cached: int) -> int:
        return sum(group.trim(seat, cached) for group in self.groups)

    def free_pages(self) -> int:
        return min((int(g.pool.num_free) for g in self.groups), default=0)

    def total_pages(self) -> int:
        return min((g.num_pages for g in self.groups), default=0)

    def pages_held(self, seat: int) -> dict[int, list[int]]:
        return {i: g.pages_of(seat) for i, g in enumerate(self.groups)}

    def bytes_per_token(self) -> int:
        extra = SCALE_BYTES if self.cache_dtype == E4M3 else 0
        return sum(g.bytes_per_token(self.cache_dtype.itemsize, extra) for g in self.groups)

    def keep_places(self, seat: int, cached: int, places) -> int:
        """Of the new tokens of a seat behind its first ``cached`` places, those at ``cached + place`` for the given places
        (rising) stay, one behind the other from ``cached`` on; the others' rows may be written over.  Returns how many
        tokens the seat holds then.  The work runs on the current stream, behind the step that wrote the rows."""
        places = [int(p) for p in places]
        if seat not in self._open:
            raise ValueError(f"seat {seat} is not open")
        if cached < 0 or any(p < 0 for p in places) or any(a >= b for a, b in zip(places, places[1:])):
            raise ValueError(f"places to keep are rising numbers from 0 on, got {places} behind {cached}")
        moved = [(cached + p, cached + i) for i, p in enumerate(places) if p != i]
        if moved and cached + places[-1] >= self.max_tokens_per_request:
            raise ValueError(f"place {cached + places[-1]} lies behind the longest request the tables hold ({self.max_tokens_per_request})")
        if moved:
            if self.state_needs:
                raise ValueError("layers with per-request state cannot take back some of a step's tokens")
            sources, targets = map(list, zip(*moved))
            found = [(group.rows_at(seat, sources), group.rows_at(seat, targets)) for group in self.groups]  # (all, before any moves)
            for group, rows in zip(self.groups, found):
                group.move_rows(*rows)
        return cached + len(places)

    # -- what a step sees -----------------------------------------------------
    def upload_tables(self, seats) -> None:
        for group in self.groups:
            group.upload(seats)

    def kv_slot(self, slot: int) -> KvSlot | None:
        group = self._group_of.get(slot)
        return group.slot_view(slot) if group is not None else None

    def state_slot(self, slot: int):
        return self.states.get(slot)
