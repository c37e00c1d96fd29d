"""What a server of many sequences does around its projections, as cases that
can be timed and checked: rotary positions, appending new keys and values to a
paged cache, and the attention of new tokens over that cache.

A paged cache is a pool of pages of `page` entries; a sequence's entry p lies
in page table[p // page] at p % page. A batch holds `tokens` new rows, those
of sequence s at offsets[s] .. offsets[s + 1] - 1; lengths[s] counts its entries
with the new ones, so its i-th new token is at position
lengths[s] - count + i and sees the entries up to itself.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPSILON = 1e-6


# ---- cases -------------------------------------------------------------------

# Frequencies: the checkpoint's (base 1e7, first 64 of 256 dimensions) and the
# usual bases and scalings of heads of 64 and 128.
def _rope(rotary, layout, theta, scaling="none", factor=1.0, original=0.0):
    return {"rotary": rotary, "layout": layout, "theta": theta, "scaling": scaling, "factor": factor,
            "original": original}


def _attend(kind, rows, cache, heads, kv, head, page, sequences, chunk, history, window=0, gated=False,
            layout="entries"):
    return {"op": "attend", "kind": kind, "rows": rows, "cache": cache, "heads": heads, "kv": kv, "head": head,
            "page": page, "sequences": sequences, "chunk": chunk, "history": history, "window": window,
            "gated": gated, "cache_layout": layout}


def listed():
    return [
        # one decode step's queries, far into a stretched context
        {"name": "rope_step", "op": "rope", "rows": "f32", "tokens": 16, "heads": 16, "head": 256,
         "last": 262143, **_rope(64, "halves", 1e7, "yarn", 4.0, 65536.0)},
        # a prompt's queries, whole heads, interleaved
        {"name": "rope_prompt", "op": "rope", "rows": "bf16", "tokens": 4099, "heads": 32, "head": 128,
         "last": 131071, **_rope(128, "pairs", 5e5, "bands", 8.0, 8192.0)},
        # one token of one sequence, the checkpoint's heads
        {"name": "append_step_1", "op": "append", "kind": "decode", "rows": "f32", "cache": "f32", "heads": 16,
         "kv": 2, "head": 256, "page": 16, "sequences": 1, "chunk": 1, "history": 1999, "norm": True,
         "cache_layout": "entries", **_rope(64, "halves", 1e7)},
        # a decode step of 32 sequences into a cache of half the size
        {"name": "append_step_32", "op": "append", "kind": "decode", "rows": "f32", "cache": "bf16", "heads": 16,
         "kv": 2, "head": 256, "page": 64, "sequences": 32, "chunk": 1, "history": 4095, "norm": True,
         "cache_layout": "entries", **_rope(64, "halves", 1e7)},
        # prompts' chunks of several sequences
        {"name": "append_chunks", "op": "append", "kind": "ragged", "rows": "bf16", "cache": "bf16", "heads": 32,
         "kv": 8, "head": 128, "page": 16, "sequences": 5, "chunk": 1021, "history": 2000, "norm": False,
         "cache_layout": "heads", **_rope(128, "halves", 5e5)},
        # one token of one sequence: latency
        {"name": "attend_step_1", **_attend("decode", "f32", "f32", 16, 2, 256, 16, 1, 1, 1999, gated=True)},
        # a decode step of 32 sequences
        {"name": "attend_step_32", **_attend("decode", "f32", "bf16", 16, 2, 256, 64, 32, 1, 4095, gated=True)},
        # few sequences, a long history
        {"name": "attend_step_long", **_attend("decode", "bf16", "bf16", 32, 8, 128, 16, 2, 1, 131071,
                                               layout="heads")},
        # a prompt's chunk of the checkpoint's benchmark, float cache
        {"name": "attend_chunk", **_attend("even", "f32", "f32", 16, 2, 256, 64, 1, 512, 3584, gated=True)},
        # continuous batching: one prompt's chunk beside 31 decoding sequences
        {"name": "attend_mixed", **_attend("mixed", "f32", "bf16", 16, 2, 256, 64, 32, 512, 3500, gated=True)},
        # prompts' chunks of several sequences
        {"name": "attend_chunks", **_attend("ragged", "bf16", "bf16", 32, 8, 128, 16, 5, 1021, 2000)},
        # a long prompt at once
        {"name": "attend_prompt", **_attend("even", "f16", "f16", 32, 4, 64, 128, 1, 8192, 0)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rope", "append", "append", "attend", "attend", "attend"))
    rows = rng.choice(("f32", "f32", "bf16", "f16"))
    cache = rng.choice(("f32", "bf16")) if rows == "f32" else rows
    head = rng.choice((64, 128, 256))
    kv = rng.choice((1, 2, 4, 8))
    heads = kv * rng.choice((1, 2, 3, 4, 6, 8))
    scaling = rng.choice(("none", "linear", "ntk", "yarn", "bands"))
    rope = _rope(rng.choice((head, head // 2, head // 4)), rng.choice(("halves", "pairs")), rng.choice((1e4, 5e5, 1e7)),
                 scaling, 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)),
                 rng.choice((4096.0, 8192.0, 65536.0)))
    if op == "rope":
        return {"op": op, "rows": rows, "tokens": _log(rng, 1, 4096), "heads": heads, "head": head,
                "last": _log(rng, 4096, 262143), **rope}
    kind = rng.choice(("decode", "decode", "ragged", "mixed", "even"))
    sequences = _log(rng, 1, 32)
    chunk = 1 if kind == "decode" else _log(rng, 2, 1024)
    history = _log(rng, 1, 60000 if kind == "decode" and sequences <= 4 else 4096)
    page = rng.choice((8, 16, 32, 64, 128, 256))
    layout = rng.choice(("entries", "heads"))
    # no more products than the long prompt, no more entries than the long histories
    while sequences * chunk * (chunk + history) * heads * head > 32 * 8192 * 4096 * 64:
        sequences, chunk, history = max(1, sequences // 2), max(1, chunk * 2 // 3), max(1, history * 2 // 3)
    while sequences * (chunk + history) * kv * head * BYTES[cache] > 200000 * 8 * 128 * 2:
        sequences, history = max(1, sequences // 2), max(1, history * 2 // 3)
    while sequences * chunk * heads * head * BYTES[rows] > 1 << 28:
        chunk //= 2
    if op == "append":
        history = min(history, 4096)
        return {"op": op, "kind": kind, "rows": rows, "cache": cache, "heads": heads, "kv": kv, "head": head,
                "page": page, "sequences": sequences, "chunk": chunk, "history": history, "norm": rng.random() < 0.5,
                "cache_layout": layout, **rope}
    window = rng.choice((0, 0, 0, _log(rng, 16, 2048)))
    return _attend(kind, rows, cache, heads, kv, head, page, sequences, chunk, history, window, rng.random() < 0.3,
                   layout)


# New tokens and entries of each sequence: a case's own, the same for every seed.
def _shape(c):
    n, chunk, history = c["sequences"], c["chunk"], c["history"]
    if c["kind"] == "decode":
        counts = [1] * n
    elif c["kind"] == "even":
        counts = [chunk] * n
    elif c["kind"] == "mixed":
        counts = [chunk] + [1] * (n - 1)
    else:  # ragged: from the whole chunk down to a seventh of it
        counts = [max(1, chunk - (6 * chunk * s) // (7 * max(n - 1, 1))) for s in range(n)]
    # histories from the longest down to a tenth of it, in no order
    past = [history - (9 * history * ((7 * s) % n)) // (10 * n) for s in range(n)]
    return counts, [p + k for p, k in zip(past, counts)]


# ---- inputs --------------------------------------------------------------------

class _State:
    pass


class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(seed)

    def normal(self, shape, kind, scale=1.0):
        t = torch.randn(shape, device=DEVICE, generator=self.g)
        return (t * scale if scale != 1.0 else t).to(TYPES[kind])


_server = None


def _library():
    """The context and the attention workspace a server opens once."""
    global _server
    if _server is None:
        from adi_amd import hip
        ctx = hip.Context(0)
        _server = hip, ctx, hip.PagedWorkspace(ctx)
    return _server


def _rope_handle(c):
    hip, ctx, _ = _library()
    return hip.Rope(ctx, c["rotary"], layout=c["layout"], theta=c["theta"], scaling=c["scaling"], factor=c["factor"],
                    original=c["original"])


def _pages(c, d, s):
    """The batch's arrays and a pool whose pages belong to the sequences in a
    random order, with a page in eight that no sequence holds."""
    counts, lengths = _shape(c)
    s.tokens, s.most, s.longest = sum(counts), max(counts), max(lengths)
    s.offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEVICE)
    s.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    held = [-(-n // c["page"]) for n in lengths]
    pool = sum(held) + sum(held) // 8 + 1
    order = torch.randperm(pool, generator=d.g, device=DEVICE).to(torch.int32)
    width = max(held)
    first = np.concatenate([[0], np.cumsum(held)])[:-1]
    at = first[:, None] + np.arange(width)[None, :]
    at = np.where(np.arange(width)[None, :] < np.array(held)[:, None], at, -1)
    at = torch.tensor(at, device=DEVICE)
    s.table = torch.where(at >= 0, order[at.clamp(min=0)], torch.full_like(at, -1, dtype=torch.int32))

    def entries():
        if c["cache_layout"] == "entries":
            return d.normal((pool, c["page"], c["kv"], c["head"]), c["cache"])
        return d.normal((pool, c["kv"], c["page"], c["head"]), c["cache"]).transpose(1, 2)

    s.keys, s.values = entries(), entries()


def prepare(case, seed):
    c, d, s = case, _Draw(seed), _State()
    s.case = c
    if c["op"] == "rope":
        s.x = d.normal((c["tokens"], c["heads"], c["head"]), c["rows"])
        s.positions = torch.randint(0, c["last"] + 1, (c["tokens"],), dtype=torch.int32, device=DEVICE, generator=d.g)
        s.out = torch.empty_like(s.x)
    else:
        _pages(c, d, s)
        if c["op"] == "append":
            s.q = d.normal((s.tokens, c["heads"], c["head"]), c["rows"])
            s.k = d.normal((s.tokens, c["kv"], c["head"]), c["rows"])
            s.v = d.normal((s.tokens, c["kv"], c["head"]), c["rows"])
            s.out = torch.empty_like(s.q)
            s.query_norm = d.normal((c["head"],), "bf16", 0.1) if c["norm"] else None
            s.key_norm = d.normal((c["head"],), "bf16", 0.1) if c["norm"] else None
        else:
            # keys of unit variance and queries of twice that: scores of a
            # deviation of two, so some entries matter far more than others
            rows = d.normal((s.tokens, c["heads"], (2 if c["gated"] else 1) * c["head"]), c["rows"], 2.0)
            s.q = rows[:, :, :c["head"]]
            s.gate = rows[:, :, c["head"]:] if c["gated"] else None
            s.out = torch.empty((s.tokens, c["heads"], c["head"]), dtype=TYPES[c["rows"]], device=DEVICE)
    if own:
        hip, ctx, _ = _library()
        if c["op"] != "attend":
            s.rope = _rope_handle(c)
        if c["op"] != "rope":
            s.cache = hip.PagedCache(ctx, s.keys, s.values)
            s.batch = hip.PagedBatch(ctx, s.offsets, s.lengths, s.table, s.tokens, s.most, s.longest)
    return s


# ---- one pass ------------------------------------------------------------------

def run(s):
    c = s.case
    if c["op"] == "rope":
        return _rope_own(s) if own else _rope_plain(s)
    if c["op"] == "append":
        return _append_own(s) if own else _append_plain(s)
    return _attend_own(s) if own else _attend_plain(s)


def _rope_own(s):
    hip, ctx, _ = _library()
    hip.rope_rows(ctx, s.rope, s.x, s.positions, s.out)
    return s.out


def _append_own(s):
    hip, ctx, _ = _library()
    hip.paged_append(ctx, s.cache, s.batch, s.k, s.v, rope=s.rope, key_norm=s.key_norm, queries=s.q,
                     query_norm=s.query_norm, queries_out=s.out)
    return {"queries": s.out, "keys": s.keys, "values": s.values}


def _attend_own(s):
    hip, ctx, workspace = _library()
    hip.paged_attention(ctx, s.cache, s.batch, s.q, s.out, workspace, window=s.case["window"], gate=s.gate)
    return s.out


# ---- plain forms: elementary torch operations in 32 bits -------------------------

def _frequencies_plain(c):
    """(radians a position [rotary / 2] in 64 bits, magnitude)."""
    r, factor = c["rotary"], c["factor"]
    theta = c["theta"]
    if c["scaling"] == "ntk":
        theta = theta * factor ** (r / (r - 2))
    i = torch.arange(r // 2, dtype=torch.float64, device=DEVICE)
    f = theta ** (-2.0 * i / r)
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "yarn":
        # dimensions that turn more than 32 times over the original context
        # stay, those that turn less than once are stretched
        def dimension(turns):
            return r * math.log(c["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(dimension(32.0)), 0), min(math.ceil(dimension(1.0)), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    if c["scaling"] == "bands":
        # wavelengths under a quarter of the original context stay, those over
        # all of it are stretched
        smooth = ((c["original"] * f / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        return f * smooth + f / factor * (1 - smooth), 1.0
    return f, 1.0


def _rotate_plain(c, x, positions):
    """x [tokens, heads, head] in 32 bits, rotated."""
    f, magnitude = _frequencies_plain(c)
    angle = positions.double()[:, None] * f[None, :]
    cosine = (torch.cos(angle) * magnitude).float()[:, None, :]
    sine = (torch.sin(angle) * magnitude).float()[:, None, :]
    r = c["rotary"]
    if c["layout"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cosine - b * sine, b * cosine + a * sine], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cosine - b * sine, b * cosine + a * sine], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _rope_plain(s):
    s.out.copy_(_rotate_plain(s.case, s.x.float(), s.positions))
    return s.out


def _rows_plain(s):
    """Each row's sequence, its place in the sequence and its position."""
    offsets, lengths = s.offsets.long(), s.lengths.long()
    row = torch.arange(s.tokens, device=DEVICE)
    sequence = torch.searchsorted(offsets[1:], row, right=True)
    place = row - offsets[sequence]
    counts = offsets[1:] - offsets[:-1]
    return sequence, place, (lengths - counts)[sequence] + place


def _norm_plain(x, weight):
    if weight is None:
        return x
    return x / (x.square().mean(-1, keepdim=True) + EPSILON).sqrt() * (1.0 + weight.float())


def _append_plain(s):
    c = s.case
    sequence, _, position = _rows_plain(s)
    s.out.copy_(_rotate_plain(c, _norm_plain(s.q.float(), s.query_norm), position))
    page = s.table.long()[sequence, position // c["page"]]
    at = position % c["page"]
    s.keys[page, at] = _rotate_plain(c, _norm_plain(s.k.float(), s.key_norm), position).to(s.keys.dtype)
    s.values[page, at] = s.v.float().to(s.values.dtype)
    return {"queries": s.out, "keys": s.keys, "values": s.values}


def _attend_plain(s):
    c = s.case
    group = c["heads"] // c["kv"]
    sequence, place, _ = _rows_plain(s)
    offsets, lengths = s.offsets.long(), s.lengths.long()
    counts = offsets[1:] - offsets[:-1]
    step = torch.arange(s.most, device=DEVICE)
    row = (offsets[:-1, None] + step).clamp(max=s.tokens - 1)
    position = (lengths - counts)[:, None] + step
    entry = torch.arange(s.longest, device=DEVICE)
    page = s.table.long()[:, entry // c["page"]].clamp(min=0)
    # [sequence, kv head, entries, head], [sequence, kv head, tokens x group, head]
    keys = s.keys[page, entry % c["page"]].permute(0, 2, 1, 3).float().contiguous()
    values = s.values[page, entry % c["page"]].permute(0, 2, 1, 3).float().contiguous()
    n, q = c["sequences"], s.most
    queries = s.q[row].float().reshape(n, q, c["kv"], group, c["head"]).permute(0, 2, 1, 3, 4)
    queries = queries.reshape(n, c["kv"], q * group, c["head"]).contiguous()
    scores = torch.matmul(queries, keys.transpose(-1, -2)) * (1.0 / math.sqrt(c["head"]))
    seen = entry <= position[..., None]
    if c["window"]:
        seen &= entry > position[..., None] - c["window"]
    seen = seen[:, None, :, None, :].expand(n, 1, q, group, s.longest).reshape(n, 1, q * group, s.longest)
    scores.masked_fill_(~seen, -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    out = torch.matmul(weights, values) / weights.sum(-1, keepdim=True)
    out = out.reshape(n, c["kv"], q, group, c["head"]).permute(0, 2, 1, 3, 4).reshape(n, q, c["heads"], c["head"])
    out = out[sequence, place]
    if s.gate is not None:
        out = out / (1.0 + torch.exp(-s.gate.float()))
    s.out.copy_(out)
    return s.out


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    c = case
    size = BYTES[c["rows"]]
    if c["op"] == "rope":
        rows = c["tokens"] * c["heads"]
        return {"bytes": 2 * rows * c["head"] * size + 4 * c["tokens"], "flops": 3 * rows * c["rotary"]}
    counts, lengths = _shape(c)
    tokens, held = sum(counts), BYTES[c["cache"]]
    if c["op"] == "append":
        rows = tokens * (c["heads"] + c["kv"])
        return {"bytes": tokens * c["head"] * (2 * c["heads"] * size + 2 * c["kv"] * (size + held)),
                "flops": rows * (3 * c["rotary"] + (4 * c["head"] if c["norm"] else 0))}
    window = c["window"] or 1 << 30
    entries, pairs = 0, 0
    for n, length in zip(counts, lengths):
        entries += min(length, n + window - 1)
        whole = np.minimum(np.arange(length - n, length) + 1, window)
        pairs += int(whole.sum())
    return {"bytes": tokens * c["heads"] * c["head"] * size * (3 if c["gated"] else 2) +
            2 * entries * c["kv"] * c["head"] * held, "flops": 4 * pairs * c["heads"] * c["head"]}


# ---- the definitions in 64 bits ------------------------------------------------------

def _exact_turn(c, x, positions):
    """Complex pairs times magnitude e^(i position frequency), x float64."""
    half = c["rotary"] // 2
    base = c["theta"]
    if c["scaling"] == "ntk":
        base *= c["factor"] ** (c["rotary"] / (c["rotary"] - 2.0))
    rate = np.array([base ** (-i / half) for i in range(half)])
    magnitude = 1.0
    if c["scaling"] == "linear":
        rate = rate / c["factor"]
    elif c["scaling"] == "yarn":
        place = [c["rotary"] * math.log(c["original"] / (2 * math.pi * t)) / (2 * math.log(base)) for t in (32.0, 1.0)]
        first, last = max(0, math.floor(place[0])), min(c["rotary"] - 1, math.ceil(place[1]))
        for i in range(half):
            part = min(1.0, max(0.0, (i - first) / max(0.001, last - first)))
            rate[i] *= (1.0 - part) + part / c["factor"]
        magnitude = 1.0 + 0.1 * math.log(c["factor"])
    elif c["scaling"] == "bands":
        for i in range(half):
            turns = c["original"] * rate[i] / (2 * math.pi)
            if turns < 1.0:
                rate[i] /= c["factor"]
            elif turns < 4.0:
                part = (turns - 1.0) / 3.0
                rate[i] = (1.0 - part) * rate[i] / c["factor"] + part * rate[i]
    angle = positions.double()[:, None, None] * torch.tensor(rate, device=DEVICE)
    wave = torch.polar(torch.full_like(angle, magnitude), angle)
    out = x.clone()
    if c["layout"] == "halves":
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * wave
        out[..., :half], out[..., half:2 * half] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:2 * half:2].contiguous(), x[..., 1:2 * half:2].contiguous()) * wave
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = z.real, z.imag
    return out


def _exact_norm(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPSILON) * (weight.double() + 1.0)


def exact(case, seed):
    global own
    held, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = held
    c = case
    if c["op"] == "rope":
        return _exact_turn(c, s.x.double(), s.positions)
    counts, lengths = _shape(c)
    table = s.table.cpu().numpy()
    first = np.concatenate([[0], np.cumsum(counts)])
    if c["op"] == "append":
        position = torch.tensor(np.concatenate([np.arange(n - k, n) for k, n in zip(counts, lengths)]), device=DEVICE)
        pages = np.concatenate([table[i, np.arange(n - k, n) // c["page"]]
                                for i, (k, n) in enumerate(zip(counts, lengths))])
        flat = torch.tensor(pages.astype(np.int64), device=DEVICE) * c["page"] + position % c["page"]
        shape = s.keys.shape
        keys = s.keys.double().reshape(-1, *shape[2:])
        values = s.values.double().reshape(-1, *shape[2:])
        keys[flat] = _exact_turn(c, _exact_norm(s.k.double(), s.key_norm), position)
        values[flat] = s.v.double()
        return {"queries": _exact_turn(c, _exact_norm(s.q.double(), s.query_norm), position),
                "keys": keys.reshape(shape), "values": values.reshape(shape)}
    group = c["heads"] // c["kv"]
    out = torch.zeros((s.tokens, c["heads"], c["head"]), dtype=torch.float64, device=DEVICE)
    for i, (count, length) in enumerate(zip(counts, lengths)):
        pages = torch.tensor(table[i, :-(-length // c["page"])].astype(np.int64), device=DEVICE)
        for h in range(c["kv"]):
            k = s.keys[pages][:, :, h].reshape(-1, c["head"])[:length].double()
            v = s.values[pages][:, :, h].reshape(-1, c["head"])[:length].double()
            # some rows at a time, so that the scores stay under 4 GB
            step = max(1, (1 << 29) // (length * group))
            for a in range(0, count, step):
                b = min(count, a + step)
                q = s.q[first[i] + a:first[i] + b, h * group:(h + 1) * group].double().reshape(-1, c["head"])
                at = torch.arange(length - count + a, length - count + b, device=DEVICE).repeat_interleave(group)
                far = at[:, None] - torch.arange(length, device=DEVICE)[None, :]
                hidden = far < 0
                if c["window"]:
                    hidden |= far >= c["window"]
                score = torch.mm(q, k.t().contiguous()) / math.sqrt(c["head"])
                score[hidden] = -math.inf
                weight = torch.softmax(score, -1)
                out[first[i] + a:first[i] + b, h * group:(h + 1) * group] = torch.mm(weight, v).reshape(
                    b - a, group, c["head"])
    if s.gate is not None:
        out *= torch.sigmoid(s.gate.double())
    return out
