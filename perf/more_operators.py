"""What a server does between two decode steps of a beam search, and with the
pages of its cache, as cases that can be timed and checked: the selection over
beams and vocabulary, states that follow their parents, page tables that are
forked, grown and given back, pages copied, and a pool compacted.

A request has `beams` rows, rows of a request lie side by side. Pages are counted:
references[p] is how many rows hold page p, 0 a free one. A row of length n
holds the pages table[row, c] of its columns c < ceil(n / page size).
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4}


# ---- cases -------------------------------------------------------------------

def _select(rows, requests, beams, vocabulary, choices, masked=0, ended=0, weights=False, settle=False):
    return {"op": "select", "rows": rows, "requests": requests, "beams": beams, "vocabulary": vocabulary,
            "choices": choices, "masked": masked, "ended": ended, "weights": weights, "settle": settle}


def _reorder(rows, requests, beams, moved, arrays, row, other=0):
    return {"op": "reorder", "rows": rows, "requests": requests, "beams": beams, "moved": moved, "arrays": arrays,
            "row": row, "other": other}


def _pages(op, cache, caches, heads, head, page, layout="entries", **more):
    return {"op": op, "cache": cache, "caches": caches, "heads": heads, "head": head, "page": page,
            "cache_layout": layout, **more}


def listed():
    return [
        # a lone request of four beams, the checkpoint's vocabulary and unused ids
        {"name": "select_1", **_select("f32", 1, 4, 248320, 8, masked=250)},
        # a step of 16 requests, some beams ended, scores by length, rows kept in place
        {"name": "select_16", **_select("f32", 16, 4, 248320, 4, masked=250, ended=1, weights=True, settle=True)},
        # many requests of wide beams, 16-bit logits
        {"name": "select_64", **_select("bf16", 64, 8, 248320, 16, masked=250)},
        # the tokens so far of 16 requests
        {"name": "reorder_tokens", **_reorder("i32", 16, 4, 2, 1, 513)},
        # the recurrent and convolution states of the checkpoint's 30 linear layers
        {"name": "reorder_states", **_reorder("f32", 4, 4, 2, 30, 524288, 24576)},
        # a step of a lone request, the checkpoint's ten attention layers
        {"name": "fork_1", **_pages("fork", "f32", 10, 2, 256, 16, requests=1, beams=4, length=2005, moved=2, new=1)},
        # a step of 32 requests into a cache of half the size
        {"name": "fork_32", **_pages("fork", "bf16", 10, 2, 256, 16, requests=32, beams=4, length=1500, moved=2, new=1)},
        # a shared prefix's last pages made a request's own
        {"name": "copy_8", **_pages("copy", "f32", 1, 2, 256, 16, pages=64, count=8, between=False, whole=False)},
        # sequences moved to another pool, heads outermost
        {"name": "copy_256", **_pages("copy", "bf16", 10, 8, 128, 64, "heads", pages=300, count=256, between=True,
                                      whole=True)},
        # a small pool after some of its sequences left
        {"name": "compact_100", **_pages("compact", "f32", 1, 2, 256, 16, pages=100, rows=4, longest=200, left=3)},
        # a server's pool, two sequences in three gone
        {"name": "compact_4096", **_pages("compact", "bf16", 10, 2, 256, 16, pages=4096, rows=60, longest=680,
                                          left=120)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("select", "select", "reorder", "fork", "fork", "copy", "compact"))
    beams = rng.choice((1, 2, 3, 4, 4, 5, 8, 8, 12, 16))
    if op == "select":
        rows = rng.choice(("f32", "f32", "bf16", "f16"))
        vocabulary = rng.choice((512, _log(rng, 1000, 248320), 248320))
        requests = _log(rng, 1, 64)
        while requests * beams * vocabulary * BYTES[rows] > 64 * 8 * 248320 * 2:
            requests = max(1, requests * 2 // 3)
        settle = rng.random() < 0.4
        choices = beams if settle else min(rng.choice((1, beams, 2 * beams, _log(rng, 1, 32))), vocabulary // 8)
        return _select(rows, requests, beams, vocabulary, choices, rng.choice((0, vocabulary // 100)),
                       rng.choice((0, 0, beams // 3)), rng.random() < 0.5, settle)
    if op == "reorder":
        beams = max(beams, 2)
        arrays, row, requests = _log(rng, 1, 40), _log(rng, 64, 524288), _log(rng, 1, 32)
        while arrays * row * requests * beams > 16 * 30 * 548864:
            arrays, requests, row = max(1, arrays * 2 // 3), max(1, requests * 2 // 3), max(64, row * 4 // 5)
        return _reorder(rng.choice(("f32", "f32", "bf16", "i32")), requests, beams, rng.randint(1, beams - 1), arrays,
                        row)
    cache = rng.choice(("f32", "bf16", "bf16", "f16"))
    heads, head, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 256)), rng.choice((8, 16, 32, 64, 128))
    layout, caches = rng.choice(("entries", "heads")), _log(rng, 1, 10)
    each = 2 * caches * heads * head * page * BYTES[cache]  # bytes of a page
    if op == "fork":
        requests, length = _log(rng, 1, 32), _log(rng, 1, 4096)
        while requests * (2 + length / page + beams * (2 + length / page / 4)) * each > 1.1e9:
            requests, length = max(1, requests * 2 // 3), max(1, length * 2 // 3)
            if requests == 1 and length < 4 * page:
                caches = max(1, caches - 1)
                each = 2 * caches * heads * head * page * BYTES[cache]
        return _pages(op, cache, caches, heads, head, page, layout, requests=requests, beams=beams, length=length,
                      moved=rng.randint(0, beams - 1), new=rng.choice((0, 1, 1, 1, 5)))
    if op == "copy":
        count = _log(rng, 1, 512)
        while count * each > 256 * 10 * 2 * 8 * 128 * 64 * 2:
            count = max(1, count * 2 // 3)
            if count == 1:
                caches = max(1, caches - 1)
                each = 2 * caches * heads * head * page * BYTES[cache]
        between = rng.random() < 0.5
        return _pages(op, cache, caches, heads, head, page, layout, pages=(1 if between else 2) * count + 5,
                      count=count, between=between, whole=rng.random() < 0.5)
    pages = _log(rng, 32, 4096)
    while pages * each > 4096 * 10 * 2 * 2 * 256 * 16 * 2:
        pages = max(16, pages * 2 // 3)
        if pages == 16:
            caches = max(1, caches - 1)
            each = 2 * caches * heads * head * page * BYTES[cache]
    rows = _log(rng, 1, max(1, min(64, pages // 8)))
    left = _log(rng, 1, max(1, min(128, pages // 8)))
    return _pages(op, cache, caches, heads, head, page, layout, pages=pages, rows=rows,
                  longest=max(1, (pages - 1 - rows - left) * page // (rows + left)), left=left)


# A fork's requests: the entries each holds, how many of them its beams share (a
# request in four has just read its prompt, and shares all), from the longest
# down to a tenth of it in no order: a case's own, the same for every seed.
def _requests(c):
    n, longest = c["requests"], c["length"]
    lengths = [max(1, longest - (9 * longest * ((7 * r) % n)) // (10 * n)) for r in range(n)]
    return [(k, k if r % 4 == 3 else 3 * k // 4 // c["page"] * c["page"]) for r, k in enumerate(lengths)]


# ---- inputs --------------------------------------------------------------------

class _State:
    pass


class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(seed)
        self.host = np.random.default_rng(seed)

    def normal(self, shape, kind, scale=1.0):
        if kind == "i32":
            return torch.randint(0, 248320, shape, dtype=torch.int32, device=DEVICE, generator=self.g)
        t = torch.randn(shape, device=DEVICE, generator=self.g)
        return (t * scale if scale != 1.0 else t).to(TYPES[kind])


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEVICE)


_server = None


def _library():
    """The context and the workspace a server opens once."""
    global _server
    if _server is None:
        from adi_amd import hip
        ctx = hip.Context(0)
        _server = hip, ctx, hip.PagedWorkspace(ctx)
    return _server


def _parents(d, requests, beams, moved):
    """Parents of a step whose survivors stay in their rows: `moved` rows of each
    request drop out and take a child of the others, in turn."""
    out = np.tile(np.arange(beams), (requests, 1))
    for r in range(requests):
        order = d.host.permutation(beams)
        for i in range(moved):
            out[r, order[i]] = order[moved + i % (beams - moved)]
    return out


def _caches(c, d, pages):
    shape = (pages, c["page"], c["heads"], c["head"])
    if c["cache_layout"] == "heads":
        shape = (pages, c["heads"], c["page"], c["head"])
    made = [d.normal(shape, c["cache"]) for _ in range(2 * c["caches"])]
    return [t.transpose(1, 2) for t in made] if c["cache_layout"] == "heads" else made


def _pool(s, caches, references):
    hip, ctx, _ = _library()
    return hip.PagedPool(ctx, [hip.PagedCache(ctx, caches[i], caches[i + 1]) for i in range(0, len(caches), 2)],
                         references, torch.zeros(1, dtype=torch.int32, device=DEVICE))


def prepare(case, seed):
    c, d, s = case, _Draw(seed), _State()
    s.case = c
    if c["op"] == "select":
        n, k, v = c["requests"], c["beams"], c["vocabulary"]
        s.logits = d.normal((n, k, v), c["rows"], 3.0)
        if c["masked"]:
            s.logits[:, :, v - c["masked"]:] = torch.finfo(TYPES[c["rows"]]).min
        # log-probabilities of some ten tokens, the beams' near each other
        s.scores = d.normal((n, 1), "f32") - 30.0 + d.normal((n, k), "f32")
        s.ended = s.weights = None
        if c["ended"]:
            order = torch.argsort(d.normal((n, k), "f32"), -1)
            s.ended = torch.zeros((n, k), dtype=torch.int32, device=DEVICE).scatter_(1, order[:, :c["ended"]], 1)
        if c["weights"]:
            s.weights = 1.0 / (12.0 + torch.randint(0, 5, (n, k), device=DEVICE, generator=d.g).float()).sqrt()
        s.out = [torch.empty((n, c["choices"]), dtype=t, device=DEVICE)
                 for t in (torch.float32, torch.int32, torch.int32)]
    elif c["op"] == "reorder":
        shape = (c["requests"], c["beams"])
        s.arrays = [d.normal((*shape, n), c["rows"]) for _ in range(c["arrays"]) for n in (c["row"], c["other"]) if n]
        s.parents = _ints(_parents(d, *shape, c["moved"]))
        if own:
            hip, ctx, _ = _library()
            s.rows = hip.StateRows(ctx, s.arrays)
    elif c["op"] == "fork":
        _prepare_fork(c, d, s)
    elif c["op"] == "copy":
        s.source = _caches(c, d, c["pages"])
        s.target = _caches(c, d, c["pages"] + 3) if c["between"] else s.source
        order = d.host.permutation(c["pages"])
        s.sources = _ints(order[:c["count"]])
        s.targets = _ints(d.host.permutation(c["pages"] + 3)[:c["count"]] if c["between"] else order[-c["count"]:])
        # the first of a page's entries, from one up, the same for every seed
        s.entries = None if c["whole"] else _ints(1 + np.arange(c["count"]) * 5 % c["page"])
        if own:
            hip, ctx, _ = _library()
            s.from_pool, s.to_pool = _pool(s, s.source, None), _pool(s, s.target, None)
    else:
        _prepare_compact(c, d, s)
    return s


def _prepare_fork(c, d, s):
    k, page, rows = c["beams"], c["page"], c["requests"] * c["beams"]
    held = _requests(c)
    longest = max(n for n, _ in held) + c["new"]
    columns = -(-longest // page)
    need = sum(-(-shared // page) + k * (-(-n // page) - -(-shared // page)) for n, shared in held)
    free = rows * (2 + c["new"] // page) + 3
    pages = need + free
    order = d.host.permutation(pages)
    table = np.full((rows, columns), -1, np.int64)
    references = np.zeros(pages, np.int64)
    parents = _parents(d, c["requests"], k, c["moved"])
    at = 0
    for r, (n, shared) in enumerate(held):
        common, whole = -(-shared // page), -(-n // page)
        table[r * k:(r + 1) * k, :common] = order[at:at + common]
        references[order[at:at + common]] = k
        at += common
        own_pages = order[at:at + k * (whole - common)].reshape(k, whole - common)
        table[r * k:(r + 1) * k, common:whole] = own_pages
        references[own_pages] = 1
        at += own_pages.size
        if shared == n:  # the first step: every row a child of the first
            parents[r] = 0
    s.caches = _caches(c, d, pages)
    s.parents, s.lengths, s.table = _ints(parents), _ints([n for n, _ in held for _ in range(k)]), _ints(table)
    s.references = _ints(references)
    # the next step's, which a user swaps with these
    s.next_lengths, s.next_table, s.next_references = s.lengths.clone(), s.table.clone(), s.references.clone()
    s.offsets = _ints(np.arange(rows + 1) * c["new"])
    s.lacking = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    if own:
        hip, ctx, _ = _library()
        s.pool = _pool(s, s.caches, s.next_references)
        s.lacking = s.pool.lacking
        s.batch = hip.PagedBatch(ctx, s.offsets, s.next_lengths, s.next_table, rows * c["new"], c["new"], longest)


def _prepare_compact(c, d, s):
    # sequences of all lengths up to the longest, `left` of them gone since
    n = c["rows"] + c["left"]
    lengths = 1 + (np.arange(n) * 7919) % c["longest"]
    need = -(-lengths // c["page"])
    assert need.sum() <= c["pages"]
    order = d.host.permutation(c["pages"])
    stays = np.sort(np.argsort((np.arange(n) * 613) % 1009, kind="stable")[:c["rows"]])
    first = np.concatenate([[0], np.cumsum(need)])
    table = np.full((c["rows"], need.max()), -1, np.int64)
    references = np.zeros(c["pages"], np.int64)
    for i, q in enumerate(stays):
        table[i, :need[q]] = order[first[q]:first[q] + need[q]]
        references[order[first[q]:first[q] + need[q]]] = 1
    s.caches = _caches(c, d, c["pages"])
    s.lengths, s.table, s.references = _ints(lengths[stays]), _ints(table), _ints(references)
    s.next_table, s.next_references = s.table.clone(), s.references.clone()
    s.live = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    if own:
        s.pool = _pool(s, s.caches, s.next_references)


# ---- one pass ------------------------------------------------------------------

def run(s):
    return {"select": _run_select, "reorder": _run_reorder, "fork": _run_fork, "copy": _run_copy,
            "compact": _run_compact}[s.case["op"]](s)


def _run_select(s):
    if own:
        hip, ctx, workspace = _library()
        hip.beam_select(ctx, s.logits, s.scores, *s.out, workspace, weights=s.weights, ended=s.ended, ended_token=7,
                        settle=s.case["settle"])
        return s.out
    return _select_plain(s)


def _run_reorder(s):
    if own:
        hip, ctx, _ = _library()
        hip.reorder_rows(ctx, s.rows, s.parents)
        return s.arrays
    return _reorder_plain(s)


def _run_fork(s):
    if own:
        hip, ctx, workspace = _library()
        hip.paged_fork(ctx, s.pool, s.batch, s.parents, workspace, lengths=s.lengths, table=s.table,
                       references=s.references)
    else:
        _fork_plain(s)
    return {"lengths": s.next_lengths, "table": s.next_table, "references": s.next_references, "lacking": s.lacking,
            "caches": s.caches}


def _run_copy(s):
    if own:
        hip, ctx, _ = _library()
        hip.paged_copy(ctx, s.from_pool, s.to_pool, s.sources, s.targets, entries=s.entries)
    else:
        _copy_plain(s.case, s.source, s.target, s.sources.long(), s.targets.long(), s.entries)
    return s.target


def _run_compact(s):
    if own:
        hip, ctx, workspace = _library()
        hip.paged_compact(ctx, s.pool, s.lengths, s.next_table, s.live, workspace, table=s.table,
                          references=s.references)
    else:
        _compact_plain(s)
    return {"table": s.next_table, "references": s.next_references, "live": s.live, "caches": s.caches}


# ---- plain forms: elementary torch operations ------------------------------------

def _select_plain(s):
    c = s.case
    n, k, v, take = c["requests"], c["beams"], c["vocabulary"], c["choices"]
    # a sum of 248,320 terms and ranks next to each other: in 64 bits
    most = s.logits.amax(-1, keepdim=True).double()
    normal = most + (s.logits.double() - most).exp_().sum(-1, keepdim=True).log()
    # a row's largest logits, the first of equal ones: by (value, last index
    # first) as one whole number
    bits = (s.logits.float() + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, ~bits & 0xFFFFFFFF, bits + 0x80000000) - 0x80000000) * v
    key += v - 1 - torch.arange(v, device=DEVICE)
    token = v - 1 - torch.topk(key, min(take, v), -1).values.remainder(v)
    score = s.scores.double()[..., None] + (s.logits.gather(-1, token).double() - normal)
    if s.ended is not None:
        gone = s.ended[..., None] != 0
        first = torch.arange(token.shape[-1], device=DEVICE) == 0
        score = torch.where(gone, torch.where(first, s.scores.double()[..., None], -math.inf), score)
        token = torch.where(gone, torch.full_like(token, 7), token)
    rank = score if s.weights is None else score * s.weights.double()[..., None]
    beam = torch.arange(k, device=DEVICE)[:, None].expand(n, k, token.shape[-1])
    rank, score, token, beam = (t.reshape(n, -1) for t in (rank, score, token, beam))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :take]
    score, token, beam = (t.gather(-1, order) for t in (score, token, beam))
    if c["settle"]:
        place = _settled_plain(beam, k)
        score, token, beam = (torch.empty_like(t).scatter_(1, place, t) for t in (score, token, beam))
    s.out[0].copy_(score)
    s.out[1].copy_(beam)
    s.out[2].copy_(token)
    return s.out


def _settled_plain(parent, k):
    """The row of each choice: the parent's for its first child, for the others the
    rows without one, ascending."""
    j = torch.arange(k, device=DEVICE)
    same = parent[:, :, None] == parent[:, None, :]
    first = ~(same & (j[None, :] < j[:, None])).any(-1)
    childless = ~(parent[:, None, :] == j[None, :, None]).any(-1)
    # rows without a child first, ascending
    rows = torch.sort((~childless).int(), dim=-1, stable=True).indices
    among = torch.cumsum((~first).int(), -1) - 1
    return torch.where(first, parent, rows.gather(-1, among.clamp(min=0)))


def _reorder_plain(s):
    request = torch.arange(s.case["requests"], device=DEVICE)[:, None]
    parents = s.parents.long()
    for t in s.arrays:
        t.copy_(t[request, parents])
    return s.arrays


def _copy_plain(c, source, target, sources, targets, entries):
    for a, b in zip(source, target):
        rows = a[sources]
        if entries is not None:
            here = torch.arange(c["page"], device=DEVICE)[None, :] < entries[:, None]
            rows = torch.where(here[..., None, None], rows, b[targets])
        b[targets] = rows


def _fork_plain(s):
    c = s.case
    k, page, new = c["beams"], c["page"], c["new"]
    rows, columns = s.table.shape
    column = torch.arange(columns, device=DEVICE)
    row = torch.arange(rows, device=DEVICE)
    parent = row // k * k + s.parents.long().reshape(-1)
    table, references = s.table.long(), s.references.long()
    length = s.lengths.long()[parent]
    table_of = table[parent]
    held = -(-length // page)
    # the last page, where it is partly filled and new entries go into it
    at = (length // page).clamp(max=columns - 1)
    last = table_of.gather(1, at[:, None])[:, 0]
    partly = (length % page > 0) & (new > 0)
    eldest = ~((parent[:, None] == parent[None, :]) & (row[None, :] < row[:, None])).any(-1)
    copies = partly & ~(eldest & (references[last.clamp(min=0)] == 1))
    wanted = -(-(length + new) // page) - held
    demand = wanted + copies.long()
    before = torch.cumsum(demand, 0) - demand
    free = torch.sort((references > 0).int(), stable=True).indices  # the free ones first, ascending
    # the page of each column of the next table
    nth = column[None, :] - held[:, None]
    fresh = (nth >= 0) & (nth < wanted[:, None])
    copied = copies[:, None] & (column[None, :] == at[:, None])
    which = before[:, None] + torch.where(copied, 0, nth + copies.long()[:, None])
    taken = free[which.clamp(0, free.numel() - 1)]
    lives = column[None, :] < (held + wanted)[:, None]
    next_table = torch.where(fresh | copied, taken, table_of)
    s.next_table.copy_(torch.where(lives, next_table, s.next_table.long()))
    s.next_lengths.copy_(length + new)
    was = column[None, :] < (-(-s.lengths.long() // page))[:, None]
    counted = references.clone()
    counted.scatter_add_(0, table.clamp(min=0).reshape(-1), -was.long().reshape(-1))
    counted.scatter_add_(0, next_table.clamp(min=0).reshape(-1), lives.long().reshape(-1))
    s.next_references.copy_(counted)
    s.lacking.copy_((demand.sum() - (references == 0).sum()).clamp(min=0)[None])
    targets = free[before.clamp(max=free.numel() - 1)]
    which = copies.nonzero()[:, 0]
    _copy_plain(c, s.caches, s.caches, last[which], targets[which], (length % page)[which])


def _compact_plain(s):
    c = s.case
    references = s.references.long()
    lives = references > 0
    live = lives.sum()
    page = torch.arange(c["pages"], device=DEVICE)
    movers = torch.nonzero(lives & (page >= live))[:, 0]
    holes = torch.nonzero(~lives & (page < live))[:, 0]
    renamed = page.clone()
    renamed[movers] = holes
    held = torch.arange(s.table.shape[1], device=DEVICE)[None, :] < (-(-s.lengths.long() // c["page"]))[:, None]
    table = s.table.long()
    s.next_table.copy_(torch.where(held, renamed[table.clamp(min=0)], table))
    counted = references.clone()
    counted[holes] = references[movers]
    counted[movers] = 0
    s.next_references.copy_(counted)
    s.live.copy_(live[None])
    _copy_plain(c, s.caches, s.caches, movers, holes, None)


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    c = case
    if c["op"] == "select":
        logits = c["requests"] * (c["beams"] - c["ended"]) * c["vocabulary"]
        small = c["requests"] * (4 * c["beams"] * (1 + bool(c["ended"]) + c["weights"]) + 12 * c["choices"])
        return {"bytes": logits * BYTES[c["rows"]] + small, "flops": 4 * logits}
    if c["op"] == "reorder":
        rows = c["requests"] * (c["moved"] + min(c["moved"], c["beams"] - c["moved"]))
        return {"bytes": rows * c["arrays"] * (c["row"] + c["other"]) * BYTES[c["rows"]] +
                4 * c["requests"] * c["beams"], "flops": 0}
    entry = 2 * c["caches"] * c["heads"] * c["head"] * BYTES[c["cache"]]
    if c["op"] == "copy":
        moved = sum(c["page"] if c["whole"] else 1 + 5 * i % c["page"] for i in range(c["count"]))
        return {"bytes": 2 * entry * moved + 8 * c["count"], "flops": 0}
    if c["op"] == "fork":
        k, page, new = c["beams"], c["page"], c["new"]
        words, copied, pages = 0, 0, 0
        for n, shared in _requests(c):
            words += k * (-(-n // page) + -(-(n + new) // page) + 3)
            pages += -(-shared // page) + k * (-(-n // page) - -(-shared // page))
            # copied and read: of rows that share all, every one's last page from
            # one, else the moved rows' from others in turn (a lone beam keeps its own)
            copies, read = ((k, 1) if k > 1 else (0, 0)) if shared == n else \
                (c["moved"], min(c["moved"], k - c["moved"]))
            copied += (copies + read) * (n % page if new else 0)
        return {"bytes": entry * copied + 4 * (words + 2 * pages), "flops": 0}
    lengths = 1 + (np.arange(c["rows"] + c["left"]) * 7919) % c["longest"]
    need = -(-lengths // c["page"])
    stays = np.argsort((np.arange(need.size) * 613) % 1009, kind="stable")[:c["rows"]]
    live = int(need[stays].sum())
    # of live pages in a random order, that part lies behind the first `live`
    moved = live * (c["pages"] - live) // c["pages"]
    return {"bytes": 2 * entry * c["page"] * moved + 8 * (live + c["pages"]), "flops": 0}


# ---- the definitions in 64 bits ------------------------------------------------------

def exact(case, seed):
    global own
    held, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = held
    return {"select": _exact_select, "reorder": _exact_reorder, "fork": _exact_fork, "copy": _exact_copy,
            "compact": _exact_compact}[case["op"]](case, s)


def _exact_select(c, s):
    """Request by request: every candidate's log-probability in 64 bits, sorted."""
    n, k, take = c["requests"], c["beams"], c["choices"]
    out = [np.zeros((n, take)), np.zeros((n, take), np.int64), np.zeros((n, take), np.int64)]
    for r in range(n):
        found = []
        for b in range(k):
            score = float(s.scores[r, b])
            weight = 1.0 if s.weights is None else float(s.weights[r, b])
            if s.ended is not None and int(s.ended[r, b]):
                found.append((-score * weight, b, 0, 7, score))
                continue
            x = s.logits[r, b].double()
            p = torch.log_softmax(x, -1)
            # a few more than are taken, all of those equal to the last one
            edge = torch.sort(x, descending=True).values[min(take, x.numel()) - 1]
            at = torch.nonzero(x >= edge)[:, 0]
            if at.numel() > 4 * take + 64:
                above = torch.nonzero(x > edge)[:, 0]
                at = torch.cat([above, torch.nonzero(x == edge)[:take, 0]])
            for t, q, l in zip(at.tolist(), p[at].tolist(), x[at].tolist()):
                found.append((-(score + q) * weight, b, -l, t, score + q))
        found.sort()
        best = found[:take]
        if c["settle"]:
            rows = [None] * take
            rest = []
            for f in best:
                if rows[f[1]] is None:
                    rows[f[1]] = f
                else:
                    rest.append(f)
            for i in range(take):
                if rows[i] is None:
                    rows[i] = rest.pop(0)
            best = rows
        for i, f in enumerate(best):
            out[0][r, i], out[1][r, i], out[2][r, i] = f[4], f[1], f[3]
    return [torch.tensor(out[0]), torch.tensor(out[1], dtype=torch.int32), torch.tensor(out[2], dtype=torch.int32)]


def _exact_reorder(c, s):
    if c["rows"] == "i32":
        return None
    parents = s.parents.cpu().numpy()
    out = []
    for t in s.arrays:
        new = torch.empty(t.shape, dtype=torch.float64, device=DEVICE)
        for r in range(c["requests"]):
            for b in range(c["beams"]):
                new[r, b] = t[r, parents[r, b]].double()
        out.append(new)
        if sum(x.numel() for x in out if x is not None) > 3e8:
            out[-1] = None  # the same operator on further arrays
    return out


def _moved(c, source, target, moves):
    """The caches after moves (from page, to page, entries), in 64 bits."""
    out = []
    for a, b in zip(source, target):
        new = b.double()
        for x, y, n in moves:
            new[y, :n] = a[x, :n].double()
        out.append(new)
        if sum(t.numel() for t in out if t is not None) > 3e8:
            out[-1] = None
    return out


def _exact_copy(c, s):
    entries = [c["page"]] * c["count"] if s.entries is None else s.entries.tolist()
    return _moved(c, s.source, s.target, list(zip(s.sources.tolist(), s.targets.tolist(), entries)))


def _exact_fork(c, s):
    """Row by row, as a server's own lists would be kept."""
    k, page, new = c["beams"], c["page"], c["new"]
    table, lengths = s.table.cpu().numpy(), s.lengths.tolist()
    held = [list(table[i, :-(-n // page)]) for i, n in enumerate(lengths)]
    count = s.references.cpu().numpy().astype(np.int64)
    free = iter([p for p in range(count.size) if count[p] == 0])
    parents = s.parents.cpu().numpy().reshape(-1)
    rows, moves, taken, seen = [], [], [], set()
    for i, p in enumerate(parents):
        q = i // k * k + int(p)
        pages, n = list(held[q]), lengths[q]
        if n % page and new and not (q not in seen and count[pages[-1]] == 1):
            to = next(free)
            moves.append((int(pages[-1]), to, n % page))
            pages[-1] = to
        seen.add(q)
        while len(pages) * page < n + new:
            pages.append(next(free))
        rows.append(pages)
        taken.append(n + new)
    after = count.copy()
    for pages in held:
        after[pages] -= 1
    for i, pages in enumerate(rows):
        for p in pages:
            after[p] += 1
        table[i, :len(pages)] = pages
    return {"lengths": _ints(taken), "table": _ints(table), "references": _ints(after), "lacking": _ints([0]),
            "caches": _moved(c, s.caches, s.caches, moves)}


def _exact_compact(c, s):
    count = s.references.cpu().numpy().astype(np.int64)
    live = int((count > 0).sum())
    holes = [p for p in range(live) if count[p] == 0]
    movers = [p for p in range(live, count.size) if count[p] > 0]
    table, lengths = s.table.cpu().numpy(), s.lengths.tolist()
    name = dict(zip(movers, holes))
    for i, n in enumerate(lengths):
        for j in range(-(-n // c["page"])):
            table[i, j] = name.get(int(table[i, j]), table[i, j])
    for x, y in name.items():
        count[y], count[x] = count[x], 0
    return {"table": _ints(table), "references": _ints(count), "live": _ints([live]),
            "caches": _moved(c, s.caches, s.caches, [(x, y, c["page"]) for x, y in name.items()])}
