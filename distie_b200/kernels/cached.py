"""The part of the CUDA kernel sets that serves caches in eight bits and steps of drafted tokens.

What is new here beside the plain operations: rows are finished from the projection and stored in one kernel whatever the
cache's type and wherever a token's place is (:meth:`CachedRows._rows_write`, csrc/cached_rows.cu); pages in eight bits are
read back for the attention of prompt portions (:meth:`CachedRows.kv_read`); single tokens and drafted tokens attend to
the cache as it is (csrc/attention_rows.cu).  :class:`~distie_b200.kernels.device.DeviceKernels` sends calls
here when the slot is in eight bits or the step's places are not its positions.
"""

from __future__ import annotations

import ctypes

import torch

from .interface import E4M3, MOST_DRAFTED, KvSlot, first_visible
from .library import KernelError, check, function

_CACHE_CODE = {torch.float32: 0, torch.bfloat16: 1, E4M3: 2}
_READ_ROWS = 256  # requests that one launch reads back


def _ptr(x):
    return x.data_ptr() if x is not None else None


def tree_splits(tiles: int, blocks: int, sms: int) -> int:
    """Shares that the keys of ``tiles`` tiles of rows, ``blocks`` blocks of 128 keys each, are cut into
    (attention_tree_tcgen05.cu): the number for which whole waves of CTAs take the least time, a CTA the time of its blocks
    and of two more for its start and end; joining the parts takes another two."""
    best, least = 1, None
    for splits in range(1, max(1, min(blocks, 64)) + 1):
        cost = -(-tiles * splits // sms) * (-(-blocks // splits) + 2) + (2 if splits > 1 else 0)
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
        if kv.k.dtype != kv.v.dtype or (kv.k.dtype != self.dtype and kv.k.dtype != E4M3):
            raise KernelError(f"{what}: a cache of {self.dtype} or {E4M3} is expected, not of {kv.k.dtype}")
        rows = (kv.num_pages, num_kv_heads, kv.page_size)
        if tuple(kv.k.shape) != (*rows, key_dim) or tuple(kv.v.shape) != (*rows, value_dim):
            raise KernelError(f"{what}: keys {(*rows, key_dim)} and values {(*rows, value_dim)} are expected, not "
                              f"{tuple(kv.k.shape)} and {tuple(kv.v.shape)}")
        if not kv.k.is_contiguous() or not kv.v.is_contiguous() or kv.block_table.dtype != torch.int32 or kv.block_table.stride(-1) != 1 \
                or kv.block_table.stride(0) != kv.block_table.shape[-1]:
            raise KernelError(f"{what}: contiguous pages and a contiguous int32 block table are expected")
        if (kv.k.dtype == E4M3) != (kv.k_scale is not None) or (kv.k_scale is None) != (kv.v_scale is None):
            raise KernelError(f"{what}: a cache in eight bits comes with the scales of its rows, and only such a cache")
        for scale in (kv.k_scale, kv.v_scale):
            if scale is not None and (scale.dtype != torch.float32 or tuple(scale.shape) != rows or not scale.is_contiguous()):
                raise KernelError(f"{what}: contiguous float32 scales {rows} are expected")
        return _CACHE_CODE[kv.k.dtype]

    # -- write ----------------------------------------------------------------------------------------------------
    def _rows_write(self, what, q, k, v, bias, step, kv, rotary, num_heads, num_kv_heads, head_dim, value_dim, q_out,
                    norm=(0, 0.0, None, None), q_temp=None) -> None:
        """q, k, v: matrices ``[T, n]`` or slices ``[S, T, n]`` of one projection (q None: no queries; v None: the values are
        the keys as projected); ``bias``: their three vectors."""
        cache_code = self._check_slot(what, kv, num_kv_heads, head_dim, value_dim)
        given = [x for x in (q, k, v) if x is not None]
        if any(x.dtype != k.dtype or x.dim() != k.dim() or x.stride(-1) != 1 for x in given) or k.dtype not in (torch.float32, self.dtype):
            raise KernelError(f"{what}: rows of float32 or {self.dtype} with unit column stride are expected")
        if k.dim() == 3 and k.dtype != torch.float32:
            raise KernelError(f"{what}: slices are float32")
        if rotary is not None and (rotary.rotary_dim > head_dim or rotary.rotary_dim % 2 or rotary.inv_freq.dtype != torch.float32
                                   or rotary.inv_freq.numel() * 2 < rotary.rotary_dim):
            raise KernelError(f"{what}: a rotary table of float32 frequencies for an even number of a head's elements is expected")
        for vector in (*bias, norm[2], norm[3]):
            if vector is not None and (vector.dtype != torch.float32 or vector.stride(-1) != 1):
                raise KernelError(f"{what}: float32 vectors are expected")
        if q_out is not None and (q_out.dtype != self.dtype or q_out.stride(-1) != 1):
            raise KernelError(f"{what}: q goes to rows of {self.dtype}")
        stride = lambda x: x.stride(-2) if x is not None else 0  # noqa: E731
        coef, every = (float(q_temp[0]), float(q_temp[1])) if q_temp else (0.0, 0.0)
        with self._here():
            check(
                function("distie_rows_write")(
                    _ptr(q), stride(q), _ptr(k), stride(k), _ptr(v), stride(v), _CACHE_CODE[k.dtype], k.shape[0] if k.dim() == 3 else 1,
                    k.stride(0) if k.dim() == 3 else 0, _ptr(bias[0]), _ptr(bias[1]), _ptr(bias[2]), int(norm[0]), float(norm[1]),
                    _ptr(norm[2]), _ptr(norm[3]), _ptr(rotary.inv_freq) if rotary is not None else None,
                    rotary.rotary_dim if rotary is not None else 0, int(rotary.interleaved) if rotary is not None else 0,
                    float(rotary.factor) if rotary is not None else 1.0, coef, every, step.positions.data_ptr(), _ptr(step.slots),
                    step.token_seq.data_ptr(), step.seq_seat.data_ptr(), kv.block_table.data_ptr(), kv.block_table.shape[-1],
                    kv.k.data_ptr(), kv.v.data_ptr(), _ptr(kv.k_scale), _ptr(kv.v_scale), step.num_tokens,
                    num_heads if q is not None else 0, num_kv_heads, head_dim, value_dim, kv.page_size, kv.num_pages, 1, _ptr(q_out),
                    stride(q_out), _CACHE_CODE[self.dtype], cache_code, self.error_flag.data_ptr(), self._stream(),
                ),
                "rows_write",
            )
        self._ran("rows_write")

    def _write_projection(self, what, qkv, bias, step, kv, rotary, num_heads, num_kv_heads, head_dim, value_dim, q_out, norm=(0, 0.0, None, None),
                          q_temp=None, values=True) -> None:
        """The same from one projection ``[q | k | v]`` (``values`` False: ``[q | k]``, the values are the keys)."""
        k0, v0 = num_heads * head_dim, (num_heads + num_kv_heads) * head_dim
        end = v0 + num_kv_heads * value_dim if values else v0
        if qkv.shape[-1] < end or (bias is not None and bias.shape[-1] < end):
            raise KernelError(f"{what}: a projection of at least {end} columns is expected, not of {qkv.shape[-1]}")
        cut = lambda x: (x[..., :k0], x[..., k0:v0], x[..., v0:end] if values else None)  # noqa: E731
        self._rows_write(what, *cut(qkv), cut(bias) if bias is not None else (None, None, None), step, kv, rotary, num_heads, num_kv_heads,
                         head_dim, value_dim, q_out, norm, q_temp)

    # -- read back ------------------------------------------------------------------------------------------------
    def kv_read(self, step, kv, window=None, chunk=None, keep_first=0) -> KvSlot:
        num_kv_heads, page = kv.k.shape[1], kv.page_size
        if kv.k_scale is None:
            raise KernelError("kv_read: the cache is in the engine's type already")
        self._check_slot("kv_read", kv, num_kv_heads, kv.k.shape[-1], kv.v.shape[-1])
        portions = step.portions
        if portions is None or len(portions) != step.num_seqs - step.num_decode_tokens:
            raise KernelError("kv_read: the step's portions (cached and new tokens of every entry of several tokens) are expected")
        keep_first = int(keep_first or 0) if window else 0
        plan, total = [], 0
        for row, (past, new) in enumerate(portions, start=step.num_decode_tokens):
            columns, seen = -(-(past + new) // page), first_visible(past, window, chunk) // page
            kept = min(seen, -(-keep_first // page))
            first = 0 if kept else seen
            plan.append((row, total, first, kept, seen if kept else kept, past + new))
            total += columns - first
        make = lambda like: torch.empty((total, num_kv_heads, page, like.shape[-1]), dtype=self.dtype, device=like.device)  # noqa: E731
        out = KvSlot(make(kv.k), make(kv.v), torch.empty_like(kv.block_table), page, total)
        for at in range(0, len(plan), _READ_ROWS):
            part = plan[at : at + _READ_ROWS]
            end = plan[at + _READ_ROWS][1] if at + _READ_ROWS < len(plan) else total
            numbers = (ctypes.c_int * (6 * len(part)))(*[n for entry in part for n in entry])
            with self._here():
                check(
                    function("distie_rows_read")(
                        numbers, len(part), kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr(),
                        kv.block_table.data_ptr(), kv.block_table.shape[-1], step.seq_seat.data_ptr(), num_kv_heads, kv.k.shape[-1],
                        kv.v.shape[-1], page, kv.num_pages, out.k.data_ptr(), out.v.data_ptr(), out.block_table.data_ptr(), part[0][1],
                        end - part[0][1], _CACHE_CODE[self.dtype], self.error_flag.data_ptr(), self._stream(),
                    ),
                    "rows_read",
                )
            self._ran("rows_read")
        return out

    # -- attention ------------------------------------------------------------------------------------------------
    def _attention_rows(self, q, out, step, kv, num_heads, num_kv_heads, head_dim, window, chunk, scale, keep_first, softcap, sink,
                        tokens: int, requests: int) -> None:
        """The first ``tokens`` tokens of the step: all of a step of drafted tokens, or its single tokens."""
        tree = step.tree
        cache_code = self._check_slot("attention", kv, num_kv_heads, head_dim, kv.v.shape[-1])
        value_dim, most = kv.v.shape[-1], 1
        if q.dtype != self.dtype or out.dtype != self.dtype or q.stride(-1) != 1 or out.stride(-1) != 1:
            raise KernelError(f"attention: queries and output of {self.dtype} with unit column stride are expected")
        if tree is not None:
            most = int(tree.most_nodes)
            if not 1 <= most <= MOST_DRAFTED or tree.bits.dtype != torch.int32 or tree.seqs.dtype != torch.int32 \
                    or tree.bits.shape[0] < tokens or not most <= 32 * tree.bits.shape[1] <= MOST_DRAFTED or not tree.bits.is_contiguous() \
                    or tuple(tree.seqs.shape) != (requests, 3) or not tree.seqs.is_contiguous():
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
        splits = max(1, min(4 * self.sm_count // blocks, step.max_kv_len // 64, 64))
        scratch = None
        if splits > 1:
            floats = function("distie_attention_rows_scratch_floats")(tokens, num_heads, value_dim, splits)
            scratch = torch.empty(floats, dtype=torch.float32, device=q.device)
        with self._here():
            check(
                function("distie_attention_rows")(
                    q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), _ptr(scratch), step.positions.data_ptr(),
                    step.token_seq.data_ptr(), step.seq_seat.data_ptr(), _ptr(tree.seqs) if tree is not None else None,
                    _ptr(tree.bits) if tree is not None else None, tree.bits.shape[1] if tree is not None else 1, requests, tokens, most,
                    kv.k.data_ptr(), kv.v.data_ptr(), _ptr(kv.k_scale), _ptr(kv.v_scale), kv.block_table.data_ptr(),
                    kv.block_table.shape[-1], num_heads, num_kv_heads, head_dim, value_dim, kv.page_size, kv.num_pages, window, chunk,
                    keep_first, float(scale), softcap, _ptr(sink), splits, _CACHE_CODE[self.dtype], cache_code,
                    self.error_flag.data_ptr(), self._stream(),
                ),
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
        splits = max(1, min(3 * self.sm_count // blocks, seen // 256, 64))
        if splits <= 12:
            splits = min(splits, 8)  # joined inside the kernel, by a cluster of CTAs
        scratch = None
        if splits > 8:
            floats = function("distie_attention_rows_scratch_floats")(tokens, num_heads, head_dim, splits)
            scratch = torch.empty(floats, dtype=torch.float32, device=q.device)
        with self._here():
            code = function("distie_attention_decode_e4m3")(
                q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), _ptr(scratch), step.positions.data_ptr(),
                step.token_seq.data_ptr(), step.seq_seat.data_ptr(), tokens, kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(),
                kv.v_scale.data_ptr(), kv.block_table.data_ptr(), kv.block_table.shape[-1], num_heads, num_kv_heads, head_dim,
                kv.page_size, kv.num_pages, window, chunk, keep_first, float(scale), softcap, _ptr(sink), splits,
                self.error_flag.data_ptr(), self._stream(),
            )
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
        scratch = None
        if splits > 1:
            floats = function("distie_attention_rows_scratch_floats")(tokens, num_heads, head_dim, splits)
            scratch = torch.empty(floats, dtype=torch.float32, device=q.device)
        with self._here():
            code = function("distie_attention_tree_tcgen05")(
                q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), _ptr(scratch), step.positions.data_ptr(),
                step.seq_seat.data_ptr(), tree.seqs.data_ptr(), tree.bits.data_ptr(), tree.bits.shape[1], requests, tokens, most,
                kv.k.data_ptr(), kv.v.data_ptr(), _ptr(kv.k_scale), _ptr(kv.v_scale), kv.block_table.data_ptr(),
                kv.block_table.shape[-1], num_heads, num_kv_heads, head_dim, kv.page_size, kv.num_pages, window, chunk, keep_first,
                float(scale), softcap, _ptr(sink), splits, self.error_flag.data_ptr(), self._stream(),
            )
        if code == -2:
            return False
        check(code, "attention_tree_tcgen05")
        self._ran("attention_tree_tcgen05", 1 if splits == 1 else 2)
        return True
