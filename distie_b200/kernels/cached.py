"""The part of the CUDA kernel sets that serves caches in eight bits and steps of drafted tokens.

What is new here beside the plain operations: rows are finished from the projection and stored in one kernel whatever the
cache's type and wherever a token's place is (:meth:`CachedRows._rows_write`, csrc/cached_rows.cu); pages in eight bits are
read back for the attention of prompt portions (:meth:`CachedRows.kv_read`); single tokens and drafted tokens attend to
the cache as it is (csrc/attention_rows.cu).  :class:`~distie_b200.kernels.device.DeviceKernels` sends calls
here when the slot is in eight bits or the step's places are not its positions.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from .interface import E4M3, MOST_DRAFTED, KvSlot, first_visible
from .library import KernelError, check, packed

_CACHE_CODE = {torch.float32: 0, torch.bfloat16: 1, E4M3: 2}
_READ_ROWS = 256  # requests that one launch reads back


def _ptr(x) -> int:
    return x.data_ptr() if x is not None else 0


@functools.lru_cache(maxsize=256)
def tree_splits(tiles: int, blocks: int, sms: int) -> int:
    """Shares that the keys of ``tiles`` tiles of rows, ``blocks`` blocks of 128 keys each, are cut into
    (attention_tree_tcgen05.cu): the number for which whole waves of CTAs, one an SM, take the least time, a CTA the time of its
    blocks and of eight more for its start and end (1.2 and 10 us); joining the parts takes another two.  (8 tiles of 24 blocks:
    45, 33, 28 and 26 us with 1 to 4 shares, 22 with 8 and 12; 64 of 17: 47, 38, 44, 44; 192 of 17: 60, 74, 80, 94.)"""
    best, least = 1, None
    for splits in range(1, max(1, min(blocks, 64)) + 1):
        cost = -(-tiles * splits // sms) * (-(-blocks // splits) + 8) + (2 if splits > 1 else 0)
        if least is None or cost < least:
            best, least = splits, cost
    return best


@functools.lru_cache(maxsize=256)
def decode_splits(blocks: int, keys: int, sms: int, wide: bool, many: bool) -> int:
    """Shares that the keys of ``blocks`` (token, group of heads) pairs are cut into (attention_decode_e4m3.cu): the number that
    takes the least time, counted in keys of a CTA that has an SM to itself.  An SM holds four CTAs of heads of 64 and three of
    128 (``wide``), one fewer with more than 8 heads each (``many``).  Two take 1.07 times as long as one, three 1.5 times (narrow
    heads 1.07), four 1.45; a CTA's start and end are 700 keys, joining up to 8 shares by a cluster of CTAs another 240, more
    than 8 by a second kernel 800.  (28 heads of 128 over 4,099 keys of 48 requests, 4 key heads: 57, 48, 56 and 52 us with 1 to 4
    shares; 1,024 keys of 64 requests: 23, 31, 30, 33.)"""
    slots = (3 if wide else 4) - many
    slower = (0.0, 1.0, 1.07, 1.5 if wide else 1.07, 1.45)
    best, least = 1, None
    for splits in range(1, max(1, min(keys // 256, 64)) + 1):
        waves, rest = divmod(blocks * splits, slots * sms)
        each = -(-keys // splits)
        cost = waves * (each * slower[slots] + 700) + (each * slower[-(-rest // sms)] + 700 if rest else 0)
        cost += 0 if splits == 1 else 240 if splits <= 8 else 800
        if least is None or cost < least:
            best, least = splits, cost
    return best


@functools.lru_cache(maxsize=256)
def rows_splits(blocks: int, keys: int, sms: int) -> int:
    """Shares that the keys of ``blocks`` tiles of 16 rows are cut into (attention_rows.cu): the number for which whole waves of
    blocks, two an SM, take the least time, a block that of its tiles of 32 keys and of one more for its start and end; joining
    the parts takes another.  (80 blocks, heads of 32: over 500 keys 45 us with one share, 23 with 3, 25 with 7; over 5,000
    356, 147 and 119.)"""
    best, least = 1, None
    for splits in range(1, max(1, min(keys // 64, 64)) + 1):
        cost = -(-blocks * splits // (2 * sms)) * (-(-keys // (32 * splits)) + 1) + (1 if splits > 1 else 0)
        if least is None or cost < least:
            best, least = splits, cost
    return best


class CachedRows:
    caches_in_8_bits = True
    drafted_tokens = True

    @staticmethod
    def _apart(step, kv) -> bool:
        """Whether new rows go to their places by the kernel here: an 8-bit slot, or places that are not the positions."""
        return kv is not None and (kv.k_scale is not None or step.slots is not None)

    def _check_slot(self, what: str, kv, num_kv_heads: int, key_dim: int, value_dim: int) -> int:
        """The slot's element type code, after a look at what the kernels take for granted."""
        k, v, table, k_scale, v_scale, device = kv.k, kv.v, kv.block_table, kv.k_scale, kv.v_scale, self.error_flag.device
        dtype, rows = k.dtype, (kv.num_pages, num_kv_heads, kv.page_size)
        if dtype != v.dtype or (dtype != self.dtype and dtype != E4M3):
            raise KernelError(f"{what}: a cache of {self.dtype} or {E4M3} is expected, not of {dtype}")
        if k.shape != (*rows, key_dim) or v.shape != (*rows, value_dim):
            raise KernelError(f"{what}: keys {(*rows, key_dim)} and values {(*rows, value_dim)} are expected, not "
                              f"{tuple(k.shape)} and {tuple(v.shape)}")
        if not (k.is_contiguous() and v.is_contiguous() and table.is_contiguous()) or table.dtype != torch.int32 or table.dim() != 2:
            raise KernelError(f"{what}: contiguous pages and a contiguous int32 block table are expected")
        if (dtype == E4M3) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise KernelError(f"{what}: a cache in eight bits comes with the scales of its rows, and only such a cache")
        if k.device != device or v.device != device or table.device != device:
            raise KernelError(f"{what}: a cache on {device} is expected")
        if k_scale is not None and not (
                k_scale.dtype == v_scale.dtype == torch.float32 and k_scale.shape == rows and v_scale.shape == rows
                and k_scale.is_contiguous() and v_scale.is_contiguous() and k_scale.device == device and v_scale.device == device):
            raise KernelError(f"{what}: contiguous float32 scales {rows} on {device} are expected")
        return _CACHE_CODE[dtype]

    def _check_slots(self, what: str, step) -> None:
        slots = step.slots
        if slots is not None and (slots.dtype != torch.int32 or slots.numel() < step.num_tokens or not slots.is_contiguous()
                                  or slots.device != self.error_flag.device):
            raise KernelError(f"{what}: an int32 place in the cache for each of {step.num_tokens} tokens is expected")

    # -- write ----------------------------------------------------------------------------------------------------
    def _rows_write(self, what, rows, bias, step, kv, rotary, num_heads, num_kv_heads, head_dim, value_dim, q_out, norm=(0, 0.0, None, None),
                    q_temp=None) -> None:
        """``rows``: (element type code, slices, elements between slices, then pointer and row stride of q, of k and of v; a null q:
        no queries, a null v: the values are the keys as projected); ``bias``: three pointers."""
        cache_code = self._check_slot(what, kv, num_kv_heads, head_dim, value_dim)
        slots, norm_kind, norm_eps, q_weight, k_weight = step.slots, *norm
        if slots is not None:
            self._check_slots(what, step)
        frequencies, rotary_dim, interleaved, rounded, factor = 0, 0, 0, 0, 1.0
        if rotary is not None:
            rotary_dim, inv_freq = rotary.rotary_dim, rotary.inv_freq
            if rotary_dim > head_dim or rotary_dim % 2 or inv_freq.dtype != torch.float32 or inv_freq.numel() * 2 < rotary_dim:
                raise KernelError(f"{what}: a rotary table of float32 frequencies for an even number of a head's elements is expected")
            frequencies, interleaved, rounded, factor = inv_freq.data_ptr(), int(rotary.interleaved), int(rotary.rounded), rotary.factor
        for vector in (q_weight, k_weight):
            if vector is not None and (vector.dtype != torch.float32 or vector.numel() != head_dim or not vector.is_contiguous()):
                raise KernelError(f"{what}: float32 weights of {head_dim} elements are expected")
        q_to = q_to_stride = 0
        if q_out is not None:
            shape, strides = q_out.shape, q_out.stride()
            if q_out.dtype != self.dtype or strides[-1] != 1 or shape[-1] < num_heads * head_dim or shape[-2] < step.num_tokens:
                raise KernelError(f"{what}: q goes to {step.num_tokens} rows of {num_heads * head_dim} elements of {self.dtype}")
            q_to, q_to_stride = q_out.data_ptr(), strides[-2]
        coef, every = (float(q_temp[0]), float(q_temp[1])) if q_temp else (0.0, 0.0)
        code, splits, split_stride, q, q_stride, k, k_stride, v, v_stride = rows
        table, k_scale, v_scale = kv.block_table, kv.k_scale, kv.v_scale
        launch, pack = packed("distie_rows_write")
        with self._here():
            check(
                launch(pack(
                    q, q_stride, k, k_stride, v, v_stride, code, splits, split_stride, *bias, norm_kind, norm_eps,
                    0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
                    frequencies, rotary_dim, interleaved, rounded, factor, coef, every, step.positions.data_ptr(),
                    0 if slots is None else slots.data_ptr(), step.token_seq.data_ptr(), step.seq_seat.data_ptr(),
                    table.data_ptr(), table.shape[1], kv.k.data_ptr(), kv.v.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
                    0 if v_scale is None else v_scale.data_ptr(), step.num_tokens, num_heads if q else 0, num_kv_heads, head_dim, value_dim,
                    kv.page_size, kv.num_pages, 1, q_to, q_to_stride, _CACHE_CODE[self.dtype], cache_code,
                    self.error_flag.data_ptr(), self._stream(),
                )),
                "rows_write",
            )
        self._ran("rows_write")

    def _write_projection(self, what, qkv, bias, step, kv, rotary, num_heads, num_kv_heads, head_dim, value_dim, q_out, norm=(0, 0.0, None, None),
                          q_temp=None, values=True) -> None:
        """From one projection ``[q | k | v]`` (``values`` False: ``[q | k]``, the values are the keys): a matrix ``[T, n]`` of
        float32 or the set's dtype, or float32 slices ``[S, T, n]``."""
        k0, v0 = num_heads * head_dim, (num_heads + num_kv_heads) * head_dim
        end = v0 + num_kv_heads * value_dim if values else v0
        dtype, shape, strides = qkv.dtype, qkv.shape, qkv.stride()
        sliced = len(shape) == 3
        if shape[-1] < end or shape[-2] < step.num_tokens or strides[-1] != 1 or (dtype != torch.float32 and (sliced or dtype != self.dtype)):
            raise KernelError(f"{what}: a projection [{step.num_tokens}, {end}] of {self.dtype} or float32, or float32 slices of one, with unit "
                              f"column stride is expected, not {tuple(shape)} of {dtype}")
        if bias is not None and (bias.dtype != torch.float32 or bias.numel() < end or not bias.is_contiguous()):
            raise KernelError(f"{what}: a float32 bias of {end} elements is expected")
        at, size, stride = qkv.data_ptr(), 4 if dtype == torch.float32 else 2, strides[-2]
        rows = (_CACHE_CODE[dtype], shape[0] if sliced else 1, strides[0] if sliced else 0, at, stride, at + k0 * size, stride,
                at + v0 * size if values else 0, stride)
        b = bias.data_ptr() if bias is not None else 0
        self._rows_write(what, rows, (b, b + 4 * k0, b + 4 * v0) if b else (0, 0, 0), step, kv, rotary, num_heads, num_kv_heads,
                         head_dim, value_dim, q_out, norm, q_temp)

    def _write_keys(self, what, k, v, step, kv) -> None:
        """Finished keys and values ``[T, n]`` of one type, any row stride."""
        num_kv_heads, key_dim, value_dim = kv.k.shape[1], kv.k.shape[-1], kv.v.shape[-1]
        if k.dtype != v.dtype or k.dtype not in (torch.float32, self.dtype) or k.stride(-1) != 1 or v.stride(-1) != 1 \
                or tuple(k.shape) != (step.num_tokens, num_kv_heads * key_dim) or tuple(v.shape) != (step.num_tokens, num_kv_heads * value_dim):
            raise KernelError(f"{what}: keys and values of one float type, a row of every kv head's for each token, are expected")
        rows = (_CACHE_CODE[k.dtype], 1, 0, 0, 0, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0))
        self._rows_write(what, rows, (0, 0, 0), step, kv, None, 0, num_kv_heads, key_dim, value_dim, None)

    # -- read back ------------------------------------------------------------------------------------------------
    def kv_read(self, step, kv, window=None, chunk=None, keep_first=0) -> KvSlot:
        k, v, table, page, pages = kv.k, kv.v, kv.block_table, kv.page_size, kv.num_pages
        if kv.k_scale is None:
            raise KernelError("kv_read: the cache is in the engine's type already")
        num_kv_heads, key_dim, value_dim = k.shape[1], k.shape[-1], v.shape[-1]
        self._check_slot("kv_read", kv, num_kv_heads, key_dim, value_dim)
        plan, total = self._read_plan(step, page, int(window or 0), int(chunk or 0), int(keep_first or 0) if window else 0)
        if key_dim == value_dim and key_dim % 8 == 0:  # (one piece of memory; the values then begin at a multiple of 16 bytes)
            k_out, v_out = torch.empty((2, total, num_kv_heads, page, key_dim), dtype=self.dtype, device=k.device).unbind()
        else:
            k_out = torch.empty((total, num_kv_heads, page, key_dim), dtype=self.dtype, device=k.device)
            v_out = torch.empty((total, num_kv_heads, page, value_dim), dtype=self.dtype, device=k.device)
        out = KvSlot(k_out, v_out, self._read_table(step, table, page, plan, (int(window or 0), int(chunk or 0), int(keep_first or 0))), page, total)
        for numbers, count, first, size in plan:
            launch, pack = packed("distie_rows_read")
            with self._here():
                check(
                    launch(pack(
                        ctypes.addressof(numbers), count, k.data_ptr(), v.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr(),
                        table.data_ptr(), table.shape[1], step.seq_seat.data_ptr(), num_kv_heads, key_dim, value_dim, page, pages,
                        k_out.data_ptr(), v_out.data_ptr(), first, size, _CACHE_CODE[self.dtype], self.error_flag.data_ptr(), self._stream(),
                    )),
                    "rows_read",
                )
            self._ran("rows_read")
        return out

    def _read_plan(self, step, page: int, window: int, chunk: int, keep_first: int):
        """(launches, pages of the result): which pages of the step's portions are read and where they go, kept with the step for
        all layers of a kind.  A launch: its rows of six numbers (see csrc/cached_rows.cu), their count, its first page, its pages."""
        key = ("read_plan", page, window, chunk, keep_first)
        made = step.derived.get(key)
        if made is None:
            portions = step.portions
            if portions is None or len(portions) != step.num_seqs - step.num_decode_tokens:
                raise KernelError("kv_read: the step's portions (cached and new tokens of every entry of several tokens) are expected")
            rows, total = [], 0
            for row, (past, new) in enumerate(portions, start=step.num_decode_tokens):
                columns, seen = -(-(past + new) // page), first_visible(past, window, chunk) // page
                kept = min(seen, -(-keep_first // page))
                first = 0 if kept else seen
                rows.append((row, total, first, kept, seen if kept else kept, past + new))
                total += columns - first
            plan = []
            for at in range(0, len(rows), _READ_ROWS):
                part = rows[at : at + _READ_ROWS]
                end = rows[at + _READ_ROWS][1] if at + _READ_ROWS < len(rows) else total
                numbers = (ctypes.c_int * (6 * len(part)))(*[n for entry in part for n in entry])
                plan.append((numbers, len(part), part[0][1], end - part[0][1]))
            made = step.derived[key] = (plan, total)
        return made

    def _read_table(self, step, table, page: int, plan, what) -> torch.Tensor:
        """The block table of the pages that ``plan`` reads back, made before any of them is read (csrc/cached_rows.cu says why) and kept
        with the step for all layers of a kind.  Into a graph it is captured with every call: a replay may bring other seats."""
        with self._here():
            capturing = table.is_cuda and torch.cuda.is_current_stream_capturing()
        key = ("read_table", page, *what, table.shape, self._stream())
        made = None if capturing else step.derived.get(key)
        if made is None:
            made = torch.empty_like(table)
            for numbers, count, _first, _size in plan:
                launch, pack = packed("distie_rows_table")
                with self._here():
                    check(launch(pack(ctypes.addressof(numbers), count, step.seq_seat.data_ptr(), page, made.data_ptr(), table.shape[1],
                                      self._stream())), "rows_table")
                self._ran("rows_table")
            if not capturing:
                step.derived[key] = made
        return made

    # -- attention ------------------------------------------------------------------------------------------------
    def _parts(self, tokens: int, num_heads: int, value_dim: int, splits: int) -> torch.Tensor:
        """Room for the parts that several shares of the keys leave: sums of values, a maximum and a sum of weights each."""
        return torch.empty(tokens * num_heads * splits * (value_dim + 2), dtype=torch.float32, device=self.error_flag.device)

    def _attention_rows(self, q, out, step, kv, num_heads, num_kv_heads, head_dim, window, chunk, scale, keep_first, softcap, sink,
                        tokens: int, requests: int) -> None:
        """The first ``tokens`` tokens of the step: all of a step of drafted tokens, or its single tokens."""
        tree = step.tree
        cache_code = self._check_slot("attention", kv, num_kv_heads, head_dim, kv.v.shape[-1])
        value_dim, most = kv.v.shape[-1], 1
        if q.dtype != self.dtype or out.dtype != self.dtype or q.stride(-1) != 1 or out.stride(-1) != 1 \
                or q.shape[0] < tokens or q.shape[-1] < num_heads * head_dim or out.shape[0] < tokens or out.shape[-1] < num_heads * value_dim:
            raise KernelError(f"attention: queries and output of {self.dtype} with unit column stride, {num_heads} heads for each of "
                              f"{tokens} tokens, are expected")
        if tokens == 0:
            return
        if tree is not None:
            most = int(tree.most_nodes)
            if not 1 <= most <= MOST_DRAFTED or tree.bits.dtype != torch.int32 or tree.seqs.dtype != torch.int32 \
                    or tree.bits.shape[0] < tokens or not most <= 32 * tree.bits.shape[1] <= MOST_DRAFTED or not tree.bits.is_contiguous() \
                    or tuple(tree.seqs.shape) != (requests, 3) or not tree.seqs.is_contiguous() \
                    or tree.bits.device != self.error_flag.device or tree.seqs.device != self.error_flag.device:
                raise KernelError(f"attention: a tree of 1 to {MOST_DRAFTED} new tokens a request with int32 masks [tokens, words] and "
                                  f"rows [{requests}, 3] is expected")
        group = num_heads // num_kv_heads
        if tree is None and self._decode_e4m3(q, out, step, kv, num_heads, num_kv_heads, head_dim, window, chunk, scale, keep_first, softcap,
                                              sink, tokens):
            return
        if tree is not None and self._tree_tcgen05(q, out, step, kv, num_heads, num_kv_heads, head_dim, window, chunk, scale, keep_first,
                                                   softcap, sink, tokens, requests, most):
            return
        blocks = requests * num_kv_heads * -(-most * group // 16)
        splits = rows_splits(blocks, max(0, step.max_kv_len - 1) // 32 * 32 + 1, self.sm_count)  # (see _decode_e4m3: lengths of as many tiles)
        scratch = self._parts(tokens, num_heads, value_dim, splits) if splits > 1 else None
        launch, pack = packed("distie_attention_rows")
        with self._here():
            check(
                launch(pack(
                    q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), _ptr(scratch), step.positions.data_ptr(),
                    step.token_seq.data_ptr(), step.seq_seat.data_ptr(), _ptr(tree.seqs) if tree is not None else 0,
                    _ptr(tree.bits) if tree is not None else 0, tree.bits.shape[1] if tree is not None else 1, requests, tokens, most,
                    kv.k.data_ptr(), kv.v.data_ptr(), _ptr(kv.k_scale), _ptr(kv.v_scale), kv.block_table.data_ptr(),
                    kv.block_table.shape[-1], num_heads, num_kv_heads, head_dim, value_dim, kv.page_size, kv.num_pages, window, chunk,
                    keep_first, float(scale), softcap, _ptr(sink), splits, _CACHE_CODE[self.dtype], cache_code,
                    self.error_flag.data_ptr(), self._stream(),
                )),
                "attention_rows",
            )
        self._ran("attention_rows", 1 if splits == 1 else 2)

    def _decode_e4m3(self, q, out, step, kv, num_heads, num_kv_heads, head_dim, window, chunk, scale, keep_first, softcap, sink,
                     tokens: int) -> bool:
        """Single tokens on the tensor cores (attention_decode_e4m3.cu); False for sizes and alignments that the kernel does not take."""
        if self.dtype != torch.bfloat16 or head_dim not in (64, 128) or kv.v.shape[-1] != head_dim:
            return False
        blocks = tokens * num_kv_heads * -(-num_heads // num_kv_heads // 16)
        seen = min(step.max_kv_len, window or chunk or step.max_kv_len)
        # (32 lengths have one number of shares: eager steps bring a new longest length every time, and the rule takes up to 40 us the
        # first time it is asked.  4 of 1,142 steps drawn over 40 to 32,000 keys have another number than by their own length.)
        splits = decode_splits(blocks, seen // 32 * 32, self.sm_count, head_dim == 128, num_heads // num_kv_heads > 8)
        scratch = self._parts(tokens, num_heads, head_dim, splits) if splits > 8 else None
        launch, pack = packed("distie_attention_decode_e4m3")
        with self._here():
            code = launch(pack(
                q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), _ptr(scratch), step.positions.data_ptr(),
                step.token_seq.data_ptr(), step.seq_seat.data_ptr(), tokens, kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(),
                kv.v_scale.data_ptr(), kv.block_table.data_ptr(), kv.block_table.shape[-1], num_heads, num_kv_heads, head_dim,
                kv.page_size, kv.num_pages, window, chunk, keep_first, float(scale), softcap, _ptr(sink), splits,
                self.error_flag.data_ptr(), self._stream(),
            ))
        if code == -2:
            return False
        check(code, "attention_decode_e4m3")
        self._ran("attention_decode_e4m3", 1 if splits <= 8 else 2)
        return True

    def _tree_tcgen05(self, q, out, step, kv, num_heads, num_kv_heads, head_dim, window, chunk, scale, keep_first, softcap, sink,
                      tokens: int, requests: int, most: int) -> bool:
        """Drafted tokens on the tensor cores (attention_tree_tcgen05.cu); False for sizes and alignments that the kernel does not take."""
        if self.dtype != torch.bfloat16 or head_dim not in (64, 128) or kv.v.shape[-1] != head_dim:
            return False
        tree, group = step.tree, num_heads // num_kv_heads
        seen = min(step.max_kv_len, (window or chunk or step.max_kv_len) + most + 128)
        splits = tree_splits(requests * num_kv_heads * -(-most * group // 128), -(-seen // 128), self.sm_count)
        scratch = self._parts(tokens, num_heads, head_dim, splits) if splits > 1 else None
        launch, pack = packed("distie_attention_tree_tcgen05")
        with self._here():
            code = launch(pack(
                q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), _ptr(scratch), step.positions.data_ptr(),
                step.token_seq.data_ptr(), step.seq_seat.data_ptr(), tree.seqs.data_ptr(), tree.bits.data_ptr(), tree.bits.shape[1], requests, tokens, most,
                kv.k.data_ptr(), kv.v.data_ptr(), _ptr(kv.k_scale), _ptr(kv.v_scale), kv.block_table.data_ptr(),
                kv.block_table.shape[-1], num_heads, num_kv_heads, head_dim, kv.page_size, kv.num_pages, window, chunk, keep_first,
                float(scale), softcap, _ptr(sink), splits, self.error_flag.data_ptr(), self._stream(),
            ))
        if code == -2:
            return False
        check(code, "attention_tree_tcgen05")
        self._ran("attention_tree_tcgen05", 1 if splits == 1 else 2)
        return True
