"""A cache of keys and values in eight bits and attention for trees of drafted tokens: what they are timed on.

Three paths.  ``cache``: a portion's projection is finished (bias, norms per head, rotation), its keys and values go into
pages of e4m3 numbers with a float32 scale a row, and everything the portion's requests hold is read back for prompt
attention.  ``single``: attention of single tokens over such a cache.  ``tree``: attention of drafted tokens, which see the
request's cached keys and their own ancestors, over a cache in 8, 16 or 32 bits.  Sizes are those of the 1.5B, 7B and 14B
layer shapes that ``bench.py`` uses and of the tests; lengths are ragged, pages are scattered over the pool.

``run`` is the plain form, in 32 bits with torch operations; with ``own`` it makes the calls that a layer makes.
``exact`` recomputes a case in 64 bits from the same seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda:0"

#: Layer shapes: heads and kv heads of 128 (heads of 64 are twice as many, heads of 32 four times).
SHAPES = {"1.5b": (12, 2), "7b": (28, 4), "14b": (40, 8)}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MOST = 448.0


# -- the cases ------------------------------------------------------------------
def listed():
    return [
        # Five tokens handed back to one short request: the smallest write, where latency is all.
        {"name": "cache_short", "path": "cache", "shape": "1.5b", "head_dim": 128, "page": 16, "requests": 1, "tokens": 5, "past": 300,
         "normed": False},
        # A whole prompt of the 14B shape with weighted norms of queries and keys.
        {"name": "cache_prompt", "path": "cache", "shape": "14b", "head_dim": 128, "page": 32, "requests": 1, "tokens": 2048, "past": 0,
         "normed": True},
        # Portions of three requests behind long pasts, odd lengths: chunked prefill in a busy batch.
        {"name": "cache_portions", "path": "cache", "shape": "7b", "head_dim": 128, "page": 16, "requests": 3, "tokens": 1733, "past": 7001,
         "normed": False},
        # One token of one request: the smallest decode step.
        {"name": "single_one", "path": "single", "shape": "1.5b", "head_dim": 128, "page": 16, "requests": 1, "past": 300, "window": 0,
         "capped": False},
        # The decode step a server spends its time in.
        {"name": "single_batch", "path": "single", "shape": "7b", "head_dim": 128, "page": 16, "requests": 8, "past": 1024, "window": 0,
         "capped": False},
        # A few requests with long contexts.
        {"name": "single_long", "path": "single", "shape": "14b", "head_dim": 128, "page": 16, "requests": 4, "past": 30011, "window": 0,
         "capped": False},
        # A large ragged batch of heads of 64 with capped scores and a sink.
        {"name": "single_wide", "path": "single", "shape": "7b", "head_dim": 64, "page": 16, "requests": 48, "past": 4099, "window": 0,
         "capped": True},
        # Five drafted tokens of one request over a cache in 16 bits.
        {"name": "tree_small", "path": "tree", "cache": "bf16", "shape": "1.5b", "head_dim": 128, "page": 16, "requests": 1, "nodes": 5,
         "past": 300, "window": 0, "capped": False},
        # The drafted tokens of a batch over a cache in 8 bits.
        {"name": "tree_batch", "path": "tree", "cache": "e4m3", "shape": "7b", "head_dim": 128, "page": 16, "requests": 8, "nodes": 26,
         "past": 2048, "window": 0, "capped": False},
        # Large trees behind long contexts in 16 bits.
        {"name": "tree_long", "path": "tree", "cache": "bf16", "shape": "14b", "head_dim": 128, "page": 32, "requests": 2, "nodes": 64,
         "past": 16001, "window": 0, "capped": False},
        # Layers with a window and a sink, heads of 64, an odd batch.
        {"name": "tree_window", "path": "tree", "cache": "e4m3", "shape": "1.5b", "head_dim": 64, "page": 16, "requests": 33, "nodes": 11,
         "past": 3000, "window": 1024, "capped": True},
        # The true 32-bit engine, heads of 32: what parity replays run.
        {"name": "tree_float32", "path": "tree", "cache": "f32", "shape": "1.5b", "head_dim": 32, "page": 8, "requests": 2, "nodes": 13,
         "past": 500, "window": 0, "capped": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_once(rng):
    path = rng.choice(["cache", "single", "single", "tree", "tree"])
    case = {"path": path, "shape": rng.choice(["1.5b", "7b", "14b"]), "head_dim": rng.choice([128, 128, 64]), "page": rng.choice([16, 16, 32, 8])}
    if path == "cache":
        case.update(requests=rng.choice([1, 1, 2, 5]), tokens=_spread(rng, 4, 4096), past=rng.choice([0, _spread(rng, 20, 9000)]),
                    normed=rng.choice([False, True]))
        case["tokens"] = max(case["tokens"], 4 * case["requests"])
        return case
    case.update(window=rng.choice([0, 0, 0, 1024]), capped=rng.choice([False, False, True]))
    if path == "single":
        case.update(requests=_spread(rng, 1, 64), past=_spread(rng, 40, 32000))
        return case
    case.update(cache=rng.choice(["bf16", "bf16", "e4m3", "e4m3", "f32"]), requests=_spread(rng, 1, 40), nodes=_spread(rng, 2, 64),
                past=_spread(rng, 20, 16000))
    if case["cache"] == "f32":
        case.update(shape="1.5b", head_dim=rng.choice([128, 64, 32]), requests=rng.choice([1, 2, 4]), nodes=_spread(rng, 2, 16),
                    past=_spread(rng, 20, 1000))
    return case


def draw(rng):
    most = max(_cost(case) for case in listed())
    while True:
        case = _draw_once(rng)
        if _cost(case) <= most:
            return case


def _cost(case):
    """About the seconds of a pass on a well used machine, to compare cases with."""
    need = work(case)
    return need["bytes"] / 4e12 + need["flops"] / 4e14


def _heads(case):
    heads, kv = SHAPES[case["shape"]]
    return heads * 128 // case["head_dim"], kv * 128 // case["head_dim"], case["head_dim"]


def _news(case):
    """New tokens of every request of the step: uneven."""
    count = case["requests"]
    if case["path"] == "single":
        return [1] * count
    if case["path"] == "tree":
        return [max(1, case["nodes"] - 3 * (i % 4)) for i in range(count)]
    weights = [1.0 + 0.7 * ((5 * i + 2) % 4) for i in range(count)]
    lengths = [max(2, int(case["tokens"] * w / sum(weights))) for w in weights]
    lengths[0] += case["tokens"] - sum(lengths)
    return lengths


def _pasts(case):
    """Cached tokens of every request, from the given number down to about half of it."""
    count, past = case["requests"], case["past"]
    return [past - past * ((7 * i) % count) // (2 * count) for i in range(count)]


def _type(case):
    return DTYPES["f32" if case.get("cache") == "f32" else "bf16"]


# -- inputs from a seed ---------------------------------------------------------
def _parents(case, seed):
    """The drafted trees: node i's parent among the nodes before it, -1 for a child of the last cached token."""
    rng = random.Random(seed * 31 + 7)
    return [[-1 if i == 0 or rng.random() < 0.1 else rng.randrange(max(0, i - 5), i) for i in range(n)] for n in _news(case)]


def _depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def _ancestors(parents):
    """Bit j of number i: node j is node i or one of its ancestors."""
    out = []
    for i, p in enumerate(parents):
        out.append((1 << i) | (out[p] if p >= 0 else 0))
    return out


def _inputs(case, seed):
    """Everything of a step on the device: the tokens' places, the block tables, the cached rows, queries or projection."""
    heads, kv_heads, dim = _heads(case)
    page, news, pasts, dtype = case["page"], _news(case), _pasts(case), _type(case)
    count, total = len(news), sum(news)
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 11)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE)  # noqa: E731
    need = [-(-(p + n) // page) for p, n in zip(pasts, news)]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed + 5)).tolist()
    table = [[order.pop() if c < n else -1 for c in range(max(need))] for n in need]
    parents = _parents(case, seed) if case["path"] == "tree" else [list(range(-1, n - 1)) for n in news]
    starts = [sum(news[:i]) for i in range(count)]
    tiles = [(s + at, min(128, n - at)) for s, n in zip(starts, news) if n > 1 for at in range(0, n, 128)]
    words = -(-max(news) // 32)
    bits = [[(a >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for p in parents for a in _ancestors(p)] if case["path"] == "tree" else [[0]]
    ints = lambda x: torch.tensor(x, dtype=torch.int64).to(torch.int32).to(DEVICE)  # noqa: E731
    made = {
        "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "pages": sum(need), "news": news, "pasts": pasts, "dtype": dtype,
        "positions": ints([p + d for p, tree in zip(pasts, parents) for d in _depths(tree)]),
        "slots": ints([p + i for p, n in zip(pasts, news) for i in range(n)]),
        "token_seq": ints([i for i, n in enumerate(news) for _ in range(n)]),
        "seq_seat": ints(list(range(count))), "table": ints(table), "tiles": ints(tiles), "num_tiles": len(tiles),
        "bits": torch.tensor(bits, dtype=torch.int64).to(DEVICE), "tree_seqs": ints([[s, n, p] for s, n, p in zip(starts, news, pasts)]),
        "window": case.get("window", 0), "scale": dim**-0.5, "softcap": 30.0 if case.get("capped") else 0.0,
        "sink": normal(heads) if case.get("capped") else None, "longest": max(p + n for p, n in zip(pasts, news)),
    }
    made["bits"] = torch.where(made["bits"] >= 1 << 31, made["bits"] - (1 << 32), made["bits"]).to(torch.int32)
    rows = (sum(need), kv_heads, page)
    if case.get("cache", "e4m3") == "e4m3":
        # Rows of e4m3 numbers that reach the type's largest one, and scales such that the values have about unit size.
        spread = torch.exp(0.4 * normal(2, *rows))
        numbers = normal(2, *rows, dim) * 110.0
        numbers = numbers.clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn)
        made.update(k=numbers[0].clone(), v=numbers[1].clone(), k_scale=(1.2 * spread[0] / 110.0).contiguous(), v_scale=(spread[1] / 110.0).contiguous())
    else:
        made.update(k=(1.2 * normal(*rows, dim)).to(dtype), v=normal(*rows, dim).to(dtype), k_scale=None, v_scale=None)
    if case["path"] == "cache":
        columns = (heads + 2 * kv_heads) * dim
        made.update(proj=1.3 * normal(total, columns), bias=0.3 * normal(columns), eps=1e-6 if case["normed"] else None,
                    q_weight=1.0 + 0.1 * normal(dim) if case["normed"] else None, k_weight=1.0 + 0.1 * normal(dim) if case["normed"] else None,
                    inv_freq=(1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float().to(DEVICE))
    else:
        made["q"] = (1.5 * normal(total, heads * dim)).to(dtype)
    return made


def prepare(case, seed):
    return _inputs(case, seed) | {"path": case["path"]}


# -- the framework's calls ------------------------------------------------------
_KERNELS: dict = {}


def _handle(state):
    """The kernel set, the step and the cache slot, as an engine holds them while it runs a step's layers."""
    from distie_b200.kernels import DraftTree, KvSlot, RotaryTable, StepTensors, make_kernels

    kernels = _KERNELS.get(state["dtype"])
    if kernels is None:
        kernels = _KERNELS[state["dtype"]] = make_kernels(state["dtype"], DEVICE)
    news, pasts = state["news"], state["pasts"]
    step = StepTensors(
        token_ids=state["positions"], positions=state["positions"], token_seq=state["token_seq"], seq_seat=state["seq_seat"],
        num_tokens=sum(news), num_seqs=len(news), num_decode_tokens=len(news) if state["path"] == "single" else 0, max_kv_len=state["longest"],
    )
    if state["path"] == "tree":
        step.slots, step.tree = state["slots"], DraftTree(state["bits"], state["tree_seqs"], max(news))
    elif state["path"] == "cache":
        step.q_tiles, step.num_q_tiles, step.portions = state["tiles"], state["num_tiles"], list(zip(pasts, news))
    slot = KvSlot(state["k"], state["v"], state["table"], state["page"], state["pages"], state["k_scale"], state["v_scale"])
    rotary = RotaryTable(state["inv_freq"], state["dim"]) if state["path"] == "cache" else None
    return kernels, step, slot, rotary


def _own(state):
    if "handle" not in state:
        state["handle"] = _handle(state)
    kernels, step, slot, rotary = state["handle"]
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    if state["path"] == "cache":
        q = torch.empty((step.num_tokens, heads * dim), dtype=state["dtype"], device=DEVICE)
        kernels.qkv_norm_write(state["proj"], state["bias"], step, slot, rotary, heads, kv_heads, dim, dim, state["eps"], state["q_weight"],
                               state["k_weight"], None, q)
        read = kernels.kv_read(step, slot)
        return q, read.k, read.v
    out = torch.empty_like(state["q"])
    kernels.attention(state["q"], out, step, slot, heads, kv_heads, dim, state["window"] or None, state["scale"], None, 0, state["softcap"],
                      state["sink"])
    return out


# -- the plain form, in 32 bits -------------------------------------------------
def _places(state):
    """The page and the row in it of every new token."""
    slots = state["slots"].long()
    seats = state["seq_seat"].long()[state["token_seq"].long()]
    return state["table"].long()[seats, slots // state["page"]], slots % state["page"]


def _normed(x, eps, weight):
    if eps is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def _turned(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _store(rows, numbers, scales, page, at):
    """Rows [tokens, kv heads, dim] as e4m3 numbers with a scale each."""
    scale = rows.abs().amax(-1) / E4M3_MOST
    unit = rows / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    numbers.view(torch.uint8)[page, :, at] = unit.clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[page, :, at] = scale


def _values(numbers, scales):
    return numbers.float() if scales is None else numbers.float() * scales[..., None]


def _read_back(state, numbers, scales):
    """The pages of all requests one behind the other; rows behind a request's last token are zeros."""
    table, page = state["table"].long(), state["page"]
    lengths = torch.tensor([p + n for p, n in zip(state["pasts"], state["news"])], device=DEVICE)
    column = torch.arange(table.shape[1], device=DEVICE)
    held = column[None, :] * page < lengths[:, None]
    rows = _values(numbers, scales)[table[held]]
    last = lengths[:, None, None] - (column[None, :, None] * page + torch.arange(page, device=DEVICE))
    return (rows * (last > 0)[held][:, None, :, None]).to(state["dtype"])


def _plain_cache(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    x = (state["proj"] + state["bias"]).reshape(-1, heads + 2 * kv_heads, dim)
    q, k, v = x[:, :heads], x[:, heads : heads + kv_heads], x[:, heads + kv_heads :]
    angles = state["positions"].double()[:, None] * state["inv_freq"].double()[None, :]
    cos, sin = angles.cos().float()[:, None, :], angles.sin().float()[:, None, :]
    q = _turned(_normed(q, state["eps"], state["q_weight"]), cos, sin)
    k = _turned(_normed(k, state["eps"], state["k_weight"]), cos, sin)
    page, at = _places(state)
    _store(k, state["k"], state["k_scale"], page, at)
    _store(v, state["v"], state["v_scale"], page, at)
    return (q.reshape(q.shape[0], -1).to(state["dtype"]), _read_back(state, state["k"], state["k_scale"]),
            _read_back(state, state["v"], state["v_scale"]))


def _padded(state):
    """Per request and place: the new token that stands there (0 past the last), and whether there is one."""
    news = torch.tensor(state["news"], device=DEVICE)
    place = torch.arange(max(state["news"]), device=DEVICE)
    there = place[None, :] < news[:, None]
    return ((news.cumsum(0) - news)[:, None] + place) * there, there


def _seen(state, token, there):
    """[requests, new tokens, keys]: what every new token sees."""
    pasts = torch.tensor(state["pasts"], device=DEVICE)
    key = torch.arange(state["table"].shape[1] * state["page"], device=DEVICE)
    position = state["positions"].long()[token]
    place = key[None, :] - pasts[:, None]  # of a key among the request's new tokens
    cached = (place < 0)[:, None, :]
    inside = (place >= 0) & (place < token.shape[1])
    spot = place.clamp(0, token.shape[1] - 1)
    if state["path"] == "tree":
        word = state["bits"][token].long()  # [requests, new tokens, words]
        index = (spot // 32)[:, None, :].expand(-1, token.shape[1], -1)
        bit = (word.gather(2, index) >> (spot % 32)[:, None, :]) & 1
        drafted = (bit == 1) & inside[:, None, :]
    else:
        drafted = inside[:, None, :].expand(-1, token.shape[1], -1)
    key_position = torch.where(place < 0, key[None, :].expand_as(place), position.gather(1, spot))
    seen = cached | drafted
    if state["window"]:
        seen = seen & (key_position[:, None, :] > position[:, :, None] - state["window"])
    return seen & there[:, :, None]


def _plain_attention(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    token, there = _padded(state)
    table = state["table"].long().clamp(min=0)
    rows = lambda numbers, scales: _values(numbers[table], None if scales is None else scales[table]).transpose(1, 2).flatten(2, 3)  # noqa: E731
    k, v = rows(state["k"], state["k_scale"]), rows(state["v"], state["v_scale"])  # [requests, kv heads, keys, dim]
    q = state["q"].float().reshape(-1, kv_heads, heads // kv_heads, dim)[token].permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).reshape(*q.shape[:4], -1) * state["scale"]
    if state["softcap"]:
        scores = state["softcap"] * torch.tanh(scores / state["softcap"])
    scores = scores.masked_fill(~_seen(state, token, there)[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    sink = None if state["sink"] is None else state["sink"].reshape(1, kv_heads, -1, 1, 1)
    if sink is not None:
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    mixed = torch.matmul(weights.flatten(2, 3), v).reshape(*q.shape) / torch.where(total > 0, total, torch.ones_like(total))
    out = mixed.permute(0, 3, 1, 2, 4)[there]
    return out.reshape(-1, heads * dim).to(state["dtype"])


def run(state):
    if own:
        return _own(state)
    return _plain_cache(state) if state["path"] == "cache" else _plain_attention(state)


# -- what a pass cannot do without ----------------------------------------------
def _pairs(case):
    """(query and key pairs that are seen, keys that some new token of their request sees), over all requests; for trees the
    drafted part is taken as half of what a chain would see."""
    pairs = keys = 0
    for past, new in zip(_pasts(case), _news(case)):
        window = case.get("window", 0)
        cached = min(past, window) if window else past
        pairs += new * cached + new * (new + 1) // 2
        keys += cached + new
    return pairs, keys


def work(case):
    heads, kv_heads, dim = _heads(case)
    tokens = sum(_news(case))
    size = _type(case).itemsize
    row = {"e4m3": dim + 4, "bf16": 2 * dim, "f32": 4 * dim}[case.get("cache", "e4m3")]
    if case["path"] == "cache":
        columns = (heads + 2 * kv_heads) * dim
        held = sum(_pasts(case)) + tokens
        moved = tokens * (columns * 4 + heads * dim * size) + 2 * kv_heads * (tokens * row + sum(_pasts(case)) * row + held * dim * size)
        return {"bytes": moved, "flops": 12 * tokens * columns + 4 * held * kv_heads * dim}
    pairs, keys = _pairs(case)
    return {"bytes": 2 * tokens * heads * dim * size + 2 * keys * kv_heads * row, "flops": 4 * pairs * heads * dim}


# -- the definition, in 64 bits -------------------------------------------------
def _exact_e4m3(x):
    """The e4m3 number nearest to x (ties to even): three bits behind the leading one, steps of 2**-9 below 2**-6."""
    size = x.abs().clamp(min=2.0**-30)
    step = torch.exp2(torch.floor(torch.log2(size)).clamp(min=-6.0) - 3.0)
    return (torch.round(x / step) * step).clamp(-E4M3_MOST, E4M3_MOST)


def _exact_rows(made, which):
    """The cached rows as 64-bit values [pages, kv heads, page, dim]."""
    scale = made[which + "_scale"]
    return made[which].double() if scale is None else made[which].double() * scale.double()[..., None]


def _exact_cache(made):
    heads, kv_heads, dim = made["heads"], made["kv_heads"], made["dim"]
    half = dim // 2
    x = made["proj"].double() + made["bias"].double()
    x = x.reshape(x.shape[0], -1, dim).clone()
    if made["eps"] is not None:
        for part, weight in ((slice(0, heads), made["q_weight"]), (slice(heads, heads + kv_heads), made["k_weight"])):
            x[:, part] = x[:, part] / ((x[:, part] ** 2).mean(-1, keepdim=True) + made["eps"]).sqrt() * weight.double()
    angle = torch.outer(made["positions"].double(), made["inv_freq"].double())[:, None, :]
    turn = torch.polar(torch.ones_like(angle), angle)
    both = heads + kv_heads
    turned = torch.complex(x[:, :both, :half], x[:, :both, half:]) * turn
    x[:, :both] = torch.cat([turned.real, turned.imag], dim=-1)
    results = [x[:, :heads].reshape(x.shape[0], -1)]
    for which, first in (("k", heads), ("v", both)):
        rows = _exact_rows(made, which)
        fresh = x[:, first : first + kv_heads]
        scale = fresh.abs().amax(-1, keepdim=True) / E4M3_MOST
        fresh = _exact_e4m3(fresh / scale) * scale
        pages, start = [], 0
        for request, (past, new) in enumerate(zip(made["pasts"], made["news"])):
            count = -(-(past + new) // made["page"])
            whole = rows[made["table"][request, :count].long()].transpose(0, 1).reshape(kv_heads, -1, dim)
            whole[:, past : past + new] = fresh[start : start + new].transpose(0, 1)
            whole[:, past + new :] = 0.0
            pages.append(whole.reshape(kv_heads, count, made["page"], dim).transpose(0, 1))
            start += new
        results.append(torch.cat(pages))
    return tuple(results)


def _exact_attention(made, parents):
    heads, kv_heads, dim = made["heads"], made["kv_heads"], made["dim"]
    out = torch.empty((sum(made["news"]), heads, dim), dtype=torch.float64, device=DEVICE)
    keys, values = made["k"], made["v"]
    start = 0
    for request, (past, new) in enumerate(zip(made["pasts"], made["news"])):
        ids = made["table"][request, : -(-(past + new) // made["page"])].long()
        held = {}
        for which in ("k", "v"):
            rows = _exact_rows({which: made[which][ids], which + "_scale": None if made[which + "_scale"] is None else made[which + "_scale"][ids]}, which)
            held[which] = rows.transpose(0, 1).reshape(kv_heads, -1, dim)[:, : past + new].repeat_interleave(heads // kv_heads, dim=0)
        seen = torch.zeros((new, past + new), dtype=torch.bool)
        seen[:, :past] = True
        depth = []
        for i in range(new):
            parent = parents[request][i]
            depth.append(depth[parent] + 1 if parent >= 0 else 0)
            if parent >= 0:
                seen[i, past:] = seen[parent, past:]
            seen[i, past + i] = True
        place = torch.tensor(list(range(past)) + [past + d for d in depth])
        if made["window"]:
            seen &= place[None, :] > place[past:, None] - made["window"]
        q = made["q"][start : start + new].double().reshape(new, heads, dim).transpose(0, 1)
        scores = q @ held["k"].transpose(1, 2) * made["scale"]
        if made["softcap"]:
            scores = torch.tanh(scores / made["softcap"]) * made["softcap"]
        scores = torch.where(seen.to(DEVICE)[None], scores, torch.full_like(scores, -math.inf))
        if made["sink"] is not None:
            scores = torch.cat([scores, made["sink"].double()[:, None, None].expand(heads, new, 1)], dim=-1)
        weights = torch.softmax(scores, dim=-1)[..., : past + new]
        out[start : start + new] = (weights @ held["v"]).transpose(0, 1)
        start += new
    return out.reshape(out.shape[0], -1)


def exact(case, seed):
    made = _inputs(case, seed)
    if case["path"] == "cache":
        return _exact_cache(made)
    parents = _parents(case, seed) if case["path"] == "tree" else [list(range(-1, n - 1)) for n in _news(case)]
    return _exact_attention(made, parents)
