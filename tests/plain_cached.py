"""Plain 64-bit versions of the operations on 8-bit caches and drafted tokens, and the steps they are tested on."""

from __future__ import annotations

import math

import torch

from distie_b200.kernels import DraftTree, KvSlot, RotaryTable, StepTensors

E4M3 = torch.float8_e4m3fn
MOST = 448.0


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def masks_of(parents):
    """Rows of booleans: node i sees node j (itself and its ancestors)."""
    n = len(parents)
    seen = torch.zeros((n, n), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def depths_of(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def random_parents(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [-1 if i == 0 else int(torch.randint(-1, i, (1,), generator=g)) for i in range(n)]


def packed(mask, words):
    """Boolean rows [n, m] as int32 words."""
    wide = torch.zeros((mask.shape[0], words * 32), dtype=torch.int64)
    wide[:, : mask.shape[1]] = mask
    bits = (wide.reshape(mask.shape[0], words, 32) << torch.arange(32)).sum(-1)
    return torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)


class Case:
    """A step of requests ``(past, parents or new tokens)`` and a cache slot with scattered pages and random rows.

    ``kind``: ``single`` (one token each), ``portion`` or ``tree``; ``cache``: a dtype.  The rows of the whole pool are
    random, those of the new tokens included; ``masks`` of a tree may be given instead of its parents' ancestors."""

    def __init__(self, kind, requests, kv_heads, dim, value_dim, page, cache, dtype, device, seed=0, masks=None, spare_pages=2):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.dim, self.value_dim, self.kv_heads, self.page = kind, dim, value_dim, kv_heads, page
        self.pasts = [p for p, _ in requests]
        self.parents = [list(r) if kind == "tree" else list(range(-1, r - 1)) for _, r in requests]
        self.news = [len(p) for p in self.parents]
        count, total = len(requests), sum(self.news)
        self.masks = masks or [masks_of(p) for p in self.parents]
        need = [max(1, -(-(p + n) // page)) for p, n in zip(self.pasts, self.news)]
        pages = sum(need) + spare_pages
        order = torch.randperm(pages, generator=g).tolist()
        seats = torch.randperm(count + 2, generator=g)[:count].tolist()  # seats in another order than the batch
        table = torch.full((count + 2, max(need) + 1), -1, dtype=torch.int32)
        for seat, n in zip(seats, need):
            table[seat, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.positions = [p + d for p, tree in zip(self.pasts, self.parents) for d in depths_of(tree)]
        self.slots = [p + i for p, n in zip(self.pasts, self.news) for i in range(n)]
        starts = [sum(self.news[:i]) for i in range(count)]
        self.starts, self.seats, self.table = starts, seats, table
        if cache == E4M3:
            make = lambda d: (torch.randn(pages, kv_heads, page, d, generator=g) * 100).clamp(-MOST, MOST).to(E4M3).to(device)  # noqa: E731
            scale = lambda: (torch.exp(torch.randn(pages, kv_heads, page, generator=g) * 0.7) / 80).to(device)  # noqa: E731
            k, v, ks, vs = make(dim), make(value_dim), scale(), scale()
        else:
            make = lambda d: torch.randn(pages, kv_heads, page, d, generator=g).to(cache).to(device)  # noqa: E731
            k, v, ks, vs = make(dim), make(value_dim), None, None
        self.kv = KvSlot(k, v, table.to(device), page, pages, ks, vs)
        tiles = [(s + at, min(128, n - at)) for s, n in zip(starts, self.news) if n > 1 for at in range(0, n, 128)]
        self.step = StepTensors(
            token_ids=ints([0] * total, device), positions=ints(self.positions, device),
            token_seq=ints([i for i, n in enumerate(self.news) for _ in range(n)], device), seq_seat=ints(seats, device),
            num_tokens=total, num_seqs=count, num_decode_tokens=0 if kind == "tree" else sum(1 for n in self.news if n == 1),
            max_kv_len=max(p + n for p, n in zip(self.pasts, self.news)),
        )
        if kind == "tree":
            words = -(-max(self.news) // 32)
            bits = torch.cat([packed(m, words) for m in self.masks]).to(device)
            self.step.slots = ints(self.slots, device)
            self.step.tree = DraftTree(bits, ints([[s, n, p] for s, n, p in zip(starts, self.news, self.pasts)], device), max(self.news))
        elif tiles:
            self.step.q_tiles, self.step.num_q_tiles = ints(tiles, device), len(tiles)
            self.step.portions = [(p, n) for p, n in zip(self.pasts, self.news) if n > 1]

    def rows(self, which):
        """The pool's rows as they are held, in 64 bits on the CPU."""
        numbers, scale = getattr(self.kv, which).double().cpu(), getattr(self.kv, which + "_scale")
        return numbers if scale is None else numbers * scale.double().cpu()[..., None]

    def held(self, which, request):
        """[kv heads, past + new, size] of a request."""
        need = -(-(self.pasts[request] + self.news[request]) // self.page)
        ids = self.table[self.seats[request], :need].long()
        rows = self.rows(which)[ids].transpose(0, 1)
        return rows.reshape(rows.shape[0], -1, rows.shape[-1])[:, : self.pasts[request] + self.news[request]]

    def seen(self, request, window=None, chunk=None, keep_first=0):
        past, new = self.pasts[request], self.news[request]
        seen = torch.ones((new, past + new), dtype=torch.bool)
        seen[:, past:] = self.masks[request]
        mine = torch.tensor(self.positions[self.starts[request] : self.starts[request] + new])
        place = torch.cat([torch.arange(past), mine])
        first = torch.zeros_like(mine)
        if window:
            first = torch.maximum(first, mine - window + 1)
        if chunk:
            first = torch.maximum(first, mine // chunk * chunk)
        return seen & ((place[None, :] >= first[:, None]) | (place[None, :] < (keep_first if window else 0)))

    def reach(self, q, heads, scale):
        """The largest sum of magnitudes behind any score, [tokens, heads * value size]: what its float32 sum is rounded relative to."""
        out = []
        for r in range(len(self.news)):
            k = self.held("k", r).repeat_interleave(heads // self.kv_heads, 0).abs()
            mine = q[self.starts[r] : self.starts[r] + self.news[r], : heads * self.dim].double().cpu().abs()
            s = mine.reshape(self.news[r], heads, self.dim).transpose(0, 1) @ k.transpose(1, 2) * scale
            out.append(s.amax(-1).transpose(0, 1).repeat_interleave(self.value_dim, 1))
        return torch.cat(out)

    def attention(self, q, heads, scale, window=None, chunk=None, keep_first=0, softcap=0.0, sink=None):
        """(output, sum of weight times magnitude of the values), 64 bits, both [tokens, heads * value size].  ``least`` then holds
        what weights in float16 may miss of an 8-bit cache's output: below 2^-14 float16 has steps of 2^-24, so every weight
        (times its value's scale, over the largest such product) may be off by 2^-25, and an element by as much of the sum of
        its numbers' magnitudes."""
        outs, sizes, least = [], [], []
        for r in range(len(self.news)):
            k, v = self.held("k", r).repeat_interleave(heads // self.kv_heads, 0), self.held("v", r).repeat_interleave(heads // self.kv_heads, 0)
            mine = q[self.starts[r] : self.starts[r] + self.news[r], : heads * self.dim].double().cpu()
            s = mine.reshape(self.news[r], heads, self.dim).transpose(0, 1) @ k.transpose(1, 2) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            seen = self.seen(r, window, chunk, keep_first)[None]
            s = s.masked_fill(~seen, -math.inf)
            column = torch.full((heads, self.news[r], 1), -math.inf, dtype=torch.float64)
            if sink is not None:
                column = sink.double().cpu().reshape(heads, 1, 1).expand(-1, self.news[r], 1)
            w = torch.softmax(torch.cat([s, column], -1), -1)[..., :-1]
            w = torch.where(seen.expand_as(w), w, torch.zeros_like(w))  # (rows that see nothing: 0 / 0)
            clean = lambda x: torch.where((w.unsqueeze(-1) > 0) | w.unsqueeze(-1).isnan(), x.unsqueeze(1), torch.zeros((), dtype=torch.float64))  # noqa: E731
            if bool(torch.isfinite(v).all()):
                out, size = w @ v, w @ v.abs()
            else:  # a value that is not finite counts for the rows that see it
                out, size = (w.unsqueeze(-1) * clean(v)).sum(2), (w.unsqueeze(-1) * clean(v.abs())).sum(2)
            small = torch.zeros_like(out)
            if self.kv.v_scale is not None:
                need = -(-(self.pasts[r] + self.news[r]) // self.page)
                ids = self.table[self.seats[r], :need].long()
                flat = lambda x: x[ids].transpose(0, 1).flatten(1, 2)[:, : v.shape[1]].repeat_interleave(heads // self.kv_heads, 0)  # noqa: E731
                most = (w * flat(self.kv.v_scale.double().cpu())[:, None]).nan_to_num(0.0).amax(-1, keepdim=True)
                small = 2.0**-25 * most * flat(self.kv.v.double().cpu()).abs().sum(1)[:, None]
            least.append(small.transpose(0, 1).reshape(self.news[r], -1))
            outs.append(out.transpose(0, 1).reshape(self.news[r], -1))
            sizes.append(size.transpose(0, 1).reshape(self.news[r], -1))
        self.least = torch.cat(least)
        return torch.cat(outs), torch.cat(sizes)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def finish(x, positions, heads, kv_heads, dim, value_dim, bias=None, rotary: RotaryTable | None = None, norm=None, q_temp=None, values=True):
    """(q, k, v) of a projection in 64 bits: [tokens, heads, size] each.  norm = (mode, eps, q weight, k weight)."""
    x = x.double().cpu()
    x = x.sum(0) if x.dim() == 3 else x
    if bias is not None:
        x = x + bias.double().cpu()
    t = x.shape[0]
    q, k = x[:, : heads * dim].reshape(t, heads, dim), x[:, heads * dim : (heads + kv_heads) * dim].reshape(t, kv_heads, dim)
    v = x[:, (heads + kv_heads) * dim : (heads + kv_heads) * dim + kv_heads * value_dim].reshape(t, kv_heads, value_dim) if values else k

    def unit(y, weight):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + norm[1])
        return y if weight is None else y * weight.double().cpu()

    def turn(y):
        if rotary is None:
            return y
        n = rotary.rotary_dim
        angle = torch.tensor(positions, dtype=torch.float64)[:, None] * rotary.inv_freq.double().cpu()[None, : n // 2]
        cos, sin = angle.cos()[:, None] * rotary.factor, angle.sin()[:, None] * rotary.factor
        y = y.clone()
        one, two = (slice(0, n, 2), slice(1, n, 2)) if rotary.interleaved else (slice(0, n // 2), slice(n // 2, n))
        a, b = y[..., one].clone(), y[..., two].clone()
        y[..., one], y[..., two] = a * cos - b * sin, b * cos + a * sin
        return y

    parts = []
    for y, weight in ((q, norm[2] if norm else None), (k, norm[3] if norm else None)):
        if norm and norm[0] == 1:
            y = unit(y, weight)
        y = turn(y)
        if norm and norm[0] == 2:
            y = unit(y, weight)
        parts.append(y)
    if q_temp:
        p = torch.tensor(positions, dtype=torch.float64)
        parts[0] = parts[0] * (1 + q_temp[0] * torch.log(torch.floor((p + 1) / q_temp[1]) + 1))[:, None, None]
    return parts[0], parts[1], v
