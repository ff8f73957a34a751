"""The plain kernel set of ``ref_kernels`` with caches in eight bits and drafted tokens: rows are finished and stored one by
one at their places, attention gathers what a token sees."""

from __future__ import annotations

import math

import torch

from distie_b200.kernels.interface import E4M3, KvSlot, first_visible
from ref_kernels import RefKernels, rotate, token_seats, whole

MOST = 448.0


def quantised(rows):
    """(e4m3 numbers, scales) of float32 rows [..., n]."""
    most = rows.abs().amax(-1)
    bad = ~torch.isfinite(rows).all(-1)
    scale = torch.where(bad, torch.full_like(most, math.nan), most / MOST)
    unit = rows / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    unit = torch.where(bad[..., None] | (scale == 0)[..., None], torch.zeros_like(unit), unit)
    return unit.clamp(-MOST, MOST).to(E4M3), scale


class RefCached(RefKernels):
    caches_in_8_bits = True
    drafted_tokens = True

    def _store(self, step, kv, k, v):
        slots = (step.slots if step.slots is not None else step.positions).long()
        pages, at = kv.block_table[token_seats(step), slots // kv.page_size].long(), slots % kv.page_size
        if bool(((pages < 0) | (pages >= kv.num_pages)).any()):
            raise IndexError("a new token's page is missing from its block table")
        for rows, numbers, scales in ((k, kv.k, kv.k_scale), (v, kv.v, kv.v_scale)):
            if scales is None:
                numbers[pages, :, at] = rows.to(numbers.dtype)
            else:
                made, scale = quantised(rows.float())
                numbers.view(torch.uint8)[pages, :, at] = made.view(torch.uint8)
                scales[pages, :, at] = scale

    def rope_kv_write(self, qkv, step, kv, rotary, num_heads, num_kv_heads, head_dim, bias=None, q_out=None):
        if kv is None or (kv.k_scale is None and step.slots is None):
            return super().rope_kv_write(qkv, step, kv, rotary, num_heads, num_kv_heads, head_dim, bias, q_out)
        finished = qkv.dim() == 2
        x = whole(qkv)
        if bias is not None and not finished:
            x = x + bias
        x = x.reshape(step.num_tokens, -1, head_dim)
        q = rotate(x[:, :num_heads], step.positions, rotary)
        k, v = rotate(x[:, num_heads : num_heads + num_kv_heads], step.positions, rotary), x[:, num_heads + num_kv_heads :]
        self._store(step, kv, k, v)
        flat = q.reshape(step.num_tokens, -1)
        if finished:
            qkv[:, : num_heads * head_dim] = flat.to(qkv.dtype)
        if q_out is not None:
            q_out.copy_(flat)

    def qkv_norm_write(self, qkv, bias, step, kv, rotary, num_heads, num_kv_heads, head_dim, value_dim, norm_eps, q_weight, k_weight, q_temp, q_out):
        if kv is None or (kv.k_scale is None and step.slots is None):
            return super().qkv_norm_write(qkv, bias, step, kv, rotary, num_heads, num_kv_heads, head_dim, value_dim, norm_eps, q_weight,
                                          k_weight, q_temp, q_out)
        super().qkv_norm_write(qkv, bias, step, None, rotary, num_heads, num_kv_heads, head_dim, value_dim, norm_eps, q_weight, k_weight, q_temp, q_out)
        x = whole(qkv) + (bias if bias is not None else 0.0)
        k0, v0 = num_heads * head_dim, (num_heads + num_kv_heads) * head_dim
        k = x[:, k0:v0].reshape(-1, num_kv_heads, head_dim)
        if norm_eps is not None:
            k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + norm_eps) * (k_weight if k_weight is not None else 1.0)
        self._store(step, kv, rotate(k, step.positions, rotary), x[:, v0 : v0 + num_kv_heads * value_dim].reshape(-1, num_kv_heads, value_dim))

    def attention(self, qkv, out, step, kv, num_heads, num_kv_heads, head_dim, window, scale, chunk=None, keep_first=0, softcap=0.0, sink=None):
        if kv.k_scale is None and step.tree is None:
            return super().attention(qkv, out, step, kv, num_heads, num_kv_heads, head_dim, window, scale, chunk, keep_first, softcap, sink)
        values = lambda numbers, scales: numbers.float() if scales is None else numbers.float() * scales[..., None]  # noqa: E731
        for t in range(step.num_tokens):
            row = int(step.token_seq[t])
            seat, position = int(step.seq_seat[row]), int(step.positions[t])
            if step.tree is not None:
                first, nodes, past = step.tree.seqs[row].tolist()
                bits = [(int(step.tree.bits[t, j // 32]) >> (j % 32)) & 1 for j in range(nodes)]
                places = [(p, p) for p in range(past)] + [(past + j, int(step.positions[first + j])) for j in range(nodes) if bits[j]]
            else:
                places = [(p, p) for p in range(position + 1)]
            oldest = first_visible(position, window, chunk)
            seen = [place for place, at in places if at >= oldest or (window and at < keep_first)]
            if not seen:
                out[t] = 0
                continue
            keys = torch.tensor(seen)
            pages, at = kv.block_table[seat, keys // kv.page_size].long(), keys % kv.page_size
            k = values(kv.k[pages, :, at], None if kv.k_scale is None else kv.k_scale[pages, :, at]).repeat_interleave(num_heads // num_kv_heads, 1)
            v = values(kv.v[pages, :, at], None if kv.v_scale is None else kv.v_scale[pages, :, at]).repeat_interleave(num_heads // num_kv_heads, 1)
            scores = torch.einsum("hd,nhd->hn", qkv[t, : num_heads * head_dim].reshape(num_heads, head_dim).float(), k) * scale
            if softcap:
                scores = softcap * torch.tanh(scores / softcap)
            if sink is not None:
                scores = torch.cat([scores, sink.reshape(-1, 1)], dim=-1)
            weights = torch.softmax(scores, dim=-1)[:, : keys.numel()]
            out[t] = torch.einsum("hn,nhd->hd", weights, v).reshape(-1).to(out.dtype)

    def kv_read(self, step, kv: KvSlot, window=None, chunk=None, keep_first=0):
        raise NotImplementedError("attention here reads the numbers as they are")
