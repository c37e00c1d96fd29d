"""Rotary positions, the paged cache's append and its attention on the GPU
against their definitions in double, at the sizes and contents where they can go
wrong: heads of every size, odd token counts, histories that end inside a page
and inside a tile, rows that see nothing, junk in pages that no row sees, page
numbers out of range, windows, strides, captured and concurrent calls.

Tolerances are worst-case bounds from the arithmetic (a rounding is off by half
a step, eps / 2 of the value), computed in double beside each result."""
import math

import numpy as np
import pytest
import torch

from adi_amd import hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of a float
PAIRS = [("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def half_step(kind):
    return torch.finfo(TYPES[kind]).eps / 2


def normal(seed, *shape, kind="f32", scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(TYPES[kind])


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def within(got, want, bound, what=""):
    """Every element within its bound; NaN and infinities in the same places."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()), float((got - want)[fine].abs().max()))


# ---- the definitions in double -------------------------------------------------

def turned(x, positions, frequencies, magnitude, layout):
    """x [tokens, heads, size] double, and the sum of the magnitudes that make
    each element (what roundings are relative to)."""
    f = torch.tensor(frequencies, dtype=torch.float64, device="cuda")
    r = 2 * f.numel()
    angle = positions.to(torch.float64)[:, None, None] * f
    c, s = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    y, size = x.clone(), x.abs()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "halves" else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * max(abs(magnitude), 1.0)
    return y, size


def rope_bound(y, size, kind):
    # the reduced angle (half a step of at most 0.79), the two sums' roundings and
    # first left-out terms, the magnitude, two products and their sum: at most
    # eight half steps of the sum of magnitudes; then the type's own rounding
    return 8 * U * size * (1 + half_step(kind)) + half_step(kind) * y.abs() + torch.finfo(TYPES[kind]).tiny


def normalized(x, weight, offset, epsilon):
    x = x.double()
    if weight is None:
        return x
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + epsilon) * (offset + weight.double())


# the sum of up to 256 squares (each lane's 8, then 6 levels, half of it through
# the root), root, quotient, weight, two products: under 16 half steps
NORM_STEPS = 16


def attention(q, keys, values, offsets, lengths, table, page, scale, window, kind, gate=None):
    """(outputs [tokens, heads, size] double, bound, rows that belong to a
    sequence). What a row does not see is left out of its sums."""
    tokens, heads, size = q.shape
    kv = keys.shape[2]
    group = heads // kv
    out = torch.zeros(tokens, heads, size, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    held = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    exact = kind == "f32"
    for s in range(len(lengths)):
        a, b, length = offsets[s], offsets[s + 1], lengths[s]
        n = b - a
        held[a:b] = True
        for i in range(n):
            p = length - n + i
            if p < 0:
                continue
            low = max(0, p - window + 1) if window else 0
            at = np.arange(low, p + 1)
            pages = torch.tensor(table[s, at // page].astype(np.int64), device="cuda")
            bad = (pages < 0) | (pages >= keys.shape[0])
            k = keys[pages.clamp(0, keys.shape[0] - 1), torch.tensor(at % page, device="cuda")].double()
            v = values[pages.clamp(0, keys.shape[0] - 1), torch.tensor(at % page, device="cuda")].double()
            k[bad], v[bad] = math.nan, math.nan
            k = k.repeat_interleave(group, 1).permute(1, 2, 0)  # [heads, size, entries]
            v = v.repeat_interleave(group, 1).permute(1, 0, 2)  # [heads, entries, size]
            x = q[a + i].double()[:, None, :]
            score = torch.bmm(x, k.contiguous())[:, 0] * scale
            sizes = torch.bmm(x.abs(), k.abs().contiguous())[:, 0].amax(-1) * scale
            w = torch.softmax(score, -1)
            o = torch.bmm(w[:, None], v)[:, 0]
            spread = torch.bmm(w[:, None], v.abs())[:, 0]
            # a score's rounding: its sum of `size` products (pieces left out: 4
            # half steps), and the exponent's roundings, relative to the
            # scores; the exponential 4 half steps
            error = sizes * (size + 8) * U + 4 * U * score.abs().amax(-1)
            weight = 2 * torch.expm1(2 * error) + 16 * U + (0 if exact else half_step(kind))
            o_bound = spread * (weight[:, None] + 3 * (at.size + 16) * U)
            if gate is not None:
                g = torch.sigmoid(gate[a + i].double())
                o, o_bound = o * g, o_bound * g + 8 * U * o.abs()
            out[a + i] = o
            bound[a + i] = o_bound + half_step(kind) * (o.abs() + o_bound) + torch.finfo(TYPES[kind]).tiny
    return out, bound, held


class Pool:
    """A pool of pages, the sequences' in a random order; `junk` fills
    what no sequence holds (whole pages, and the entries behind each length)."""

    def __init__(self, seed, lengths, page, kv, size, kind, heads_first=False, spare=3, junk=math.nan, wide=0):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((max(len(lengths), 1), max(max(need, default=0), 1) + wide), -1, np.int64)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (pages, kv, page, size) if heads_first else (pages, page, kv, size)
        self.keys, self.values = normal(seed + 1, *shape, kind=kind), normal(seed + 2, *shape, kind=kind)
        if heads_first:
            self.keys, self.values = self.keys.transpose(1, 2), self.values.transpose(1, 2)
        if junk is not None:
            for pool in (self.keys, self.values):
                unheld = torch.ones(pages, page, dtype=torch.bool, device="cuda")
                for s, n in enumerate(lengths):
                    for p in range(need[s]):
                        unheld[int(self.table[s, p]), :min(page, n - p * page)] = False
                pool[unheld] = junk
        self.page, self.lengths = page, list(lengths)

    def batch(self, gpu, counts, tokens=None, max_tokens=None, max_length=None):
        self.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(int)
        self.tokens = int(self.offsets[-1]) if tokens is None else tokens
        return hip.PagedBatch(gpu, ints(self.offsets), ints(self.lengths), ints(self.table), self.tokens,
                              max(counts) if max_tokens is None else max_tokens,
                              max(self.lengths) if max_length is None else max_length)

    def cache(self, gpu):
        return hip.PagedCache(gpu, self.keys, self.values)


@pytest.fixture(scope="module")
def workspace(gpu):
    w = hip.PagedWorkspace(gpu)
    yield w
    gpu.synchronize()
    w.close()


# ---- rotary positions -----------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("tokens,heads,size,rotary", [
    (1, 16, 256, 64), (3, 1, 64, 64), (129, 5, 128, 32), (7, 3, 80, 20), (5, 2, 97, 6), (2, 2, 1024, 1024),
    (65, 4, 2, 2)])
def test_rope_rows(gpu, kind, layout, tokens, heads, size, rotary):
    rope = hip.Rope(gpu, rotary, layout, 1e6, "yarn", 4.0, 4096.0)
    f, m = hip.rope_frequencies(rotary, layout, 1e6, "yarn", 4.0, 4096.0)
    x = normal(tokens * size, tokens, heads, size, kind=kind)
    positions = torch.randint(0, 262144, (tokens,), dtype=torch.int32, device="cuda")
    positions[0] = 0
    positions[-1] = 262143
    out = torch.empty_like(x)
    hip.rope_rows(gpu, rope, x, positions, out)
    want, sizes = turned(x.double(), positions, f, m, layout)
    within(out, want, rope_bound(want, sizes, kind))
    hip.rope_rows(gpu, rope, x, positions, x)  # in place
    assert torch.equal(x, out)


def test_rope_strides_far_positions_and_untouched_elements(gpu):
    """Rows inside larger arrays at addresses that are no multiple of 16 bytes,
    positions up to 2^32 - 1, and nothing else written."""
    rope = hip.Rope(gpu, 32, "halves", 1e4)
    f, m = hip.rope_frequencies(32, "halves", 1e4)
    for shift in (0, 1, 4):
        whole = normal(7, 9, 5, 103, kind="bf16")
        x = whole[:, 1:4, shift:shift + 64]
        keep = whole.clone()
        positions = ints([0, 1, 2, 1 << 20, (1 << 31) - 1, -1, -7, -(1 << 31), 5])
        want, sizes = turned(x.double(), positions.to(torch.int64) & 0xFFFFFFFF, f, m, "halves")
        out = torch.full((9, 3, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
        hip.rope_rows(gpu, rope, x, positions, out[:, :, 1])
        # an angle of 2^32 radians is held to 2^-20 in 64 bits, here and there
        within(out[:, :, 1], want, rope_bound(want, sizes, "bf16") + 2.0 ** -19 * sizes)
        assert bool((out[:, :, 0] == 3.0).all())
        hip.rope_rows(gpu, rope, x, positions, x)
        assert torch.equal(x, out[:, :, 1])
        keep[:, 1:4, shift:shift + 64] = out[:, :, 1]
        assert torch.equal(whole, keep)


def test_rope_many_tokens_and_none(gpu):
    rope = hip.Rope(gpu, 2, "pairs", 1e4)
    n = (1 << 18) + 1000  # more tokens than blocks
    x = normal(3, n, 1, 2)
    out = torch.empty_like(x)
    positions = torch.arange(n, dtype=torch.int32, device="cuda")
    hip.rope_rows(gpu, rope, x, positions, out)
    want, sizes = turned(x.double(), positions, [1.0], 1.0, "pairs")
    within(out, want, rope_bound(want, sizes, "f32"))
    hip.rope_rows(gpu, rope, x[:0], positions[:0], out[:0])


def test_rope_refusals(gpu):
    rope = hip.Rope(gpu, 64)
    x = normal(1, 2, 2, 64)
    p = ints([0, 1])
    for args in [(normal(1, 2, 2, 32), p, normal(1, 2, 2, 32)),           # fewer dimensions than rotary
                 (x, p, torch.empty(2, 2, 64, dtype=torch.float16, device="cuda")),
                 (x, p, torch.empty(2, 3, 64, device="cuda")),
                 (x, p[:1], torch.empty_like(x)),
                 (x, p.long(), torch.empty_like(x)),
                 (x, p.cpu(), torch.empty_like(x)),
                 (x.cpu(), p, torch.empty_like(x)),
                 (x.double(), p, x.double()),
                 (x[:1].expand(2, 2, 64), p, torch.empty_like(x)),
                 (x, p, x.as_strided((2, 2, 64), (64, 128, 1))),           # another layout of the same memory
                 (x.transpose(1, 2), p, x)]:
        with pytest.raises(hip.HipError) as info:
            hip.rope_rows(gpu, rope, *args)
        assert info.value.status == hip.INVALID_ARGUMENT
    with pytest.raises(hip.HipError, match="rotary"):
        hip.Rope(gpu, 63)
    rope.close()
    with pytest.raises(hip.HipError, match="null"):
        hip.rope_rows(gpu, rope, x, p, x)


# ---- append ---------------------------------------------------------------------

def check_append(gpu, rows, kind, size, heads, kv, page, counts, lengths, layout="halves", rotary=None, norm=True,
                 queries=True, heads_first=False, padding=0, in_place=False):
    pool = Pool(size + page, lengths, page, kv, size, kind, heads_first, junk=None)
    batch = pool.batch(gpu, counts, tokens=sum(counts) + padding)
    n = pool.tokens
    q, k, v = (normal(50 + i, n, h, size, kind=rows) for i, h in enumerate((heads, kv, kv)))
    weight = [normal(60 + i, size, kind="bf16", scale=0.1) if norm else None for i in range(2)]
    rope = hip.Rope(gpu, rotary, layout, 1e5) if rotary else None
    f, m = hip.rope_frequencies(rotary, layout, 1e5) if rotary else ([], 1.0)
    keys, values = pool.keys.clone(), pool.values.clone()
    q_in = q.clone()
    q_out = q if in_place else torch.full_like(q, 5.0)
    hip.paged_append(gpu, pool.cache(gpu), batch, k, v, rope, weight[0], q if queries else None, weight[1],
                     None if in_place or not queries else q_out, weight_offset=1.0, epsilon=1e-6)
    positions = np.full(n, 0)
    written = torch.zeros(keys.shape[:2], dtype=torch.bool, device="cuda")
    owned = np.zeros(n, bool)
    for s, (a, b, length) in enumerate(zip(pool.offsets, pool.offsets[1:], lengths)):
        owned[a:b] = True
        for t in range(a, b):
            positions[t] = max(length - (b - a) + t - a, 0)
    position = torch.tensor(positions, device="cuda")
    steps = NORM_STEPS if norm else 0

    def want_of(x, w, out_kind):
        x = normalized(x, w, 1.0, 1e-6)
        y, sizes = turned(x, position, f, m, layout) if rotary else (x, x.abs())
        return y, rope_bound(y, sizes * (1 + steps * U), out_kind) + steps * U * sizes * (1 + half_step(out_kind))

    wk, bk = want_of(k, weight[0], kind)
    wv = v.to(TYPES[kind])
    for s, (a, b, length) in enumerate(zip(pool.offsets, pool.offsets[1:], lengths)):
        for t in range(a, b):
            p = length - (b - a) + t - a
            if p < 0:
                continue
            at = int(pool.table[s, p // page]), p % page
            written[at] = True
            within(pool.keys[at], wk[t], bk[t], (s, t))
            assert torch.equal(pool.values[at], wv[t])
    assert torch.equal(pool.keys[~written], keys[~written])
    assert torch.equal(pool.values[~written], values[~written])
    if queries:
        wq, bq = want_of(q_in, weight[1], rows)
        own = torch.tensor(owned, device="cuda")
        within(q_out[own], wq[own], bq[own])
        assert torch.equal(q_out[~own], q_in[~own] if in_place else torch.full_like(q[~own], 5.0))


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_append_types_sizes_layouts(gpu, rows, kind, size, layout):
    check_append(gpu, rows, kind, size, 6, 3, 16, [1, 5, 17], [1, 40, 17], layout, size // 2)


@pytest.mark.parametrize("rotary", [None, 2, 6, 20, 64])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_append_rotary_dimensions(gpu, rotary, norm, layout):
    check_append(gpu, "bf16", "bf16", 64, 2, 1, 8, [9, 1], [9, 100], layout, rotary, norm)


@pytest.mark.parametrize("counts,lengths", [
    ([1], [1]), ([0, 1, 0], [5, 9, 0]), ([3, 2], [2, 0]), ([1] * 70, list(range(1, 71))), ([200], [200]),
    ([0], [0])])
def test_append_batches(gpu, counts, lengths):
    """Sequences without rows, more rows than entries (padding in front),
    more sequences than a wave's lanes, a whole prompt; rows of no sequence."""
    check_append(gpu, "f32", "bf16", 128, 8, 2, 32, counts, lengths, "halves", 128, padding=3)


def test_append_variants(gpu):
    check_append(gpu, "f32", "f32", 256, 16, 2, 64, [4], [130], "halves", 64, heads_first=True)
    check_append(gpu, "f32", "f32", 256, 16, 2, 64, [4], [130], "halves", 64, queries=False)
    check_append(gpu, "f16", "f16", 64, 32, 8, 4096, [6, 2], [4100, 9], "pairs", 64, in_place=True, padding=2)


def test_append_bad_pages_and_bounds(gpu):
    """Entries of pages that are not the pool's are not written, a sequence
    over the batch's bounds is appended nowhere and its queries are NaN, and
    the other sequences are as ever."""
    lengths, counts = [20, 20, 20], [4, 4, 4]
    pool = Pool(5, lengths, 8, 2, 64, "f32", junk=None)
    pool.table[0, 2] = pool.keys.shape[0]  # entries 16 .. 19
    before = pool.keys.clone(), pool.values.clone()
    batch = pool.batch(gpu, counts)
    q, k, v = normal(1, 12, 2, 64), normal(2, 12, 2, 64), normal(3, 12, 2, 64)
    out = torch.empty_like(q)
    hip.paged_append(gpu, pool.cache(gpu), batch, k, v, queries=q, queries_out=out)
    assert torch.equal(out, q)
    want = before[0].clone()
    for s in (1, 2):
        want[int(pool.table[s, 2]), :4] = k[4 * s:4 * s + 4]
    assert torch.equal(pool.keys, want)
    # lengths and offsets that the host's bounds do not cover
    pool.keys.copy_(before[0])
    over = hip.PagedBatch(gpu, ints([0, 4, 8, 12]), ints([20, 25, 20]), ints(pool.table), 12, 4, 24)
    hip.paged_append(gpu, pool.cache(gpu), over, k, v, queries=q, queries_out=out)
    assert bool(torch.isnan(out[4:8]).all()) and torch.equal(out[:4], q[:4]) and torch.equal(out[8:], q[8:])
    want = before[0].clone()
    want[int(pool.table[2, 2]), :4] = k[8:]
    assert torch.equal(pool.keys, want)
    pool.keys.copy_(before[0])
    many = hip.PagedBatch(gpu, ints([0, 5, 8, 1000]), ints([20, 20, 20]), ints(pool.table), 12, 4, 24)
    hip.paged_append(gpu, pool.cache(gpu), many, k, v, queries=q, queries_out=out)
    assert bool(torch.isnan(out[:5]).all()) and torch.equal(out[5:], q[5:])


# ---- attention --------------------------------------------------------------------

def check_attention(gpu, workspace, rows, kind, size, heads, kv, page, counts, lengths, window=0, gated=False,
                    heads_first=False, padding=0, scale=0.0, junk=math.nan, seed=11, query_scale=2.0, bend=None,
                    max_tokens=None, max_length=None):
    pool = Pool(seed, lengths, page, kv, size, kind, heads_first, junk=junk)
    batch = pool.batch(gpu, counts, tokens=sum(counts) + padding, max_tokens=max_tokens, max_length=max_length)
    n = pool.tokens
    both = normal(seed + 3, n, heads, 2 * size, kind=rows, scale=query_scale)
    q, gate = both[..., :size], both[..., size:] if gated else None
    if bend is not None:
        bend(pool, q)
    out = torch.full((n, heads, size), 7.0, dtype=TYPES[rows], device="cuda")
    hip.paged_attention(gpu, pool.cache(gpu), batch, q, out, workspace, scale=scale, window=window, gate=gate)
    want, bound, held = attention(q, pool.keys, pool.values, pool.offsets, lengths, pool.table, page,
                                  scale or 1 / math.sqrt(size), window, rows, gate)
    within(out[held], want[held], bound[held])
    assert bool((out[~held] == 7.0).all())
    return out


SHAPES = [  # heads, KV heads, new tokens, lengths
    (2, 1, [1], [1]),
    (16, 2, [1], [33]),
    (8, 8, [1, 1, 1], [64, 17, 300]),
    (6, 2, [5, 1, 3], [5, 129, 260]),       # up to 15 rows a KV head
    (8, 1, [3, 17, 1], [40, 17, 333]),      # more
    (5, 1, [60], [60]),
    (16, 2, [40, 1, 1, 9], [300, 700, 31, 9]),
]


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_types_and_shapes(gpu, workspace, rows, kind, size, shape):
    heads, kv, counts, lengths = SHAPES[shape]
    check_attention(gpu, workspace, rows, kind, size, heads, kv, [8, 16, 64][shape % 3], counts, lengths,
                    gated=shape % 2 == 0, heads_first=shape % 3 == 1)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("window", [1, 7, 32, 100, 5000])
@pytest.mark.parametrize("counts,lengths", [([1, 1], [200, 3]), ([3], [300]), ([70, 2], [250, 90])])
def test_attention_windows(gpu, workspace, rows, kind, window, counts, lengths):
    check_attention(gpu, workspace, rows, kind, 64, 4, 2, 16, counts, lengths, window=window)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("heads", [4, 64])
def test_attention_rows_that_see_nothing(gpu, workspace, rows, kind, heads):
    """Front padding, empty sequences, sequences without rows, rows behind
    the last sequence."""
    check_attention(gpu, workspace, rows, kind, 64, heads, 2, 16, [3, 0, 2, 4], [1, 50, 0, 40], padding=5)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("heads,counts,lengths", [
    (2, [4], [37]), (2, [7, 2], [70, 100]), (32, [4], [37]), (16, [40, 3], [90, 35])])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("window", [0, 20])
def test_attention_infinities_in_entries_some_rows_do_not_see(gpu, workspace, rows, kind, heads, counts, lengths, value,
                                                           window):
    """A value or key that is not finite in an entry among the new ones: the rows
    before it (and past its window) are as if it was not there."""
    for which in ("values", "keys"):
        pool = Pool(21, lengths, 16, 2, 64, kind)
        batch = pool.batch(gpu, counts)
        q = normal(5, pool.tokens, heads, 64, kind=rows)
        out = torch.empty_like(q)
        hip.paged_attention(gpu, pool.cache(gpu), batch, q, out, workspace, window=window)
        for s, (n, length) in enumerate(zip(counts, lengths)):
            at = length - n + 1  # the second new token's entry
            page = int(pool.table[s, at // 16])
            getattr(pool, which)[page, at % 16, :, 3] = value
        got = torch.empty_like(q)
        hip.paged_attention(gpu, pool.cache(gpu), batch, q, got, workspace, window=window)
        for s, (a, b) in enumerate(zip(pool.offsets, pool.offsets[1:])):
            assert torch.equal(got[a], out[a]), (which, s)
            if b - a < 2:
                continue
            seen = b - a if window == 0 else min(b - a, 1 + window)
            if which == "values":
                assert not bool(torch.isfinite(got[a + 1:a + seen, :, 3]).any())
                rest = [i for i in range(64) if i != 3]
                assert torch.equal(got[a + 1:a + seen][..., rest], out[a + 1:a + seen][..., rest])
            if seen < b - a:
                assert torch.equal(got[a + seen:b], out[a + seen:b])


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 3, 1]])
def test_attention_bad_pages(gpu, workspace, rows, kind, counts):
    """A page number that is not the pool's: the rows that see its entries are
    NaN, the others are as ever; entries before a window may have no page."""
    lengths = [100, 50, 200]

    def bend(pool, q):
        pool.table[0, 5] = pool.keys.shape[0]       # entries 80 .. 95
        pool.table[2, 0] = -1                       # entries 0 .. 15

    pool = Pool(31, lengths, 16, 2, 64, kind)
    bend(pool, None)
    batch = pool.batch(gpu, counts)
    q = normal(6, pool.tokens, 8, 64, kind=rows)
    for window in (0, 60):
        out = torch.empty_like(q)
        hip.paged_attention(gpu, pool.cache(gpu), batch, q, out, workspace, window=window)
        want, bound, _ = attention(q, pool.keys, pool.values, pool.offsets, lengths, pool.table, 16, 1 / 8, window,
                                   rows)
        within(out, want, bound)
        assert bool(torch.isnan(out[0]).any()) == (counts[0] == 1 or 60 + 0 >= 80)
        assert bool(torch.isnan(out[-1]).any()) == (window == 0)


@pytest.mark.parametrize("heads", [4, 64])
def test_attention_bounds(gpu, workspace, heads):
    """A sequence over the batch's bounds is NaN, the others are as ever."""
    counts, lengths = [2, 2, 2], [40, 50, 30]
    pool = Pool(8, lengths, 16, 2, 128, "bf16")
    q = normal(9, 6, heads, 128, kind="bf16")
    out, got = torch.empty_like(q), torch.empty_like(q)
    hip.paged_attention(gpu, pool.cache(gpu), pool.batch(gpu, counts), q, out, workspace)
    hip.paged_attention(gpu, pool.cache(gpu), pool.batch(gpu, counts, max_length=45), q, got, workspace)
    assert torch.equal(got[:2], out[:2]) and bool(torch.isnan(got[2:4]).all()) and torch.equal(got[4:], out[4:])
    many = hip.PagedBatch(gpu, ints([0, 2, 5, 6]), ints(lengths), ints(pool.table), 6, 2, 50)
    hip.paged_attention(gpu, pool.cache(gpu), many, q, got, workspace)
    assert torch.equal(got[:2], out[:2]) and bool(torch.isnan(got[2:5]).all()) and bool(torch.isfinite(got[5]).all())


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("scale,query_scale", [(1.0, 30.0), (1e-3, 1.0), (0.0, 1e3)])
def test_attention_scores_near_and_far(gpu, workspace, rows, kind, scale, query_scale):
    """Weights that are nearly one entry's, and nearly even."""
    if rows != "f32" and query_scale > 100:
        query_scale = 100.0
    for counts, lengths in (([1], [700]), ([33], [300])):
        check_attention(gpu, workspace, rows, kind, 64, 4, 2, 32, counts, lengths, scale=scale, query_scale=query_scale)


@pytest.mark.parametrize("rows,kind", PAIRS)
def test_attention_floats_of_every_size(gpu, workspace, rows, kind):
    """Values and queries far from one: no piece of a float is lost."""
    if rows == "f16":
        pytest.skip("f16 has no such range")

    def bend(pool, q):
        pool.values.mul_(2.0 ** 60)
        pool.keys.mul_(2.0 ** -60)
        q.mul_(2.0 ** 60)

    for counts, lengths in (([1], [100]), ([33], [100])):
        check_attention(gpu, workspace, rows, kind, 64, 4, 2, 32, counts, lengths, bend=bend)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("counts,lengths", [([1, 1], [3000, 900]), ([2], [5000]), ([40, 1], [2000, 1500])])
def test_attention_long_histories(gpu, workspace, rows, kind, counts, lengths):
    """Histories in parts, whole in a workspace that holds few of them, and
    with a looser host bound than needed (other parts)."""
    a = check_attention(gpu, workspace, rows, kind, 128, 16, 2, 64, counts, lengths)
    small = hip.PagedWorkspace(gpu, 1 << 20)
    b = check_attention(gpu, small, rows, kind, 128, 16, 2, 64, counts, lengths)
    assert (a.double() - b.double()).abs().max() <= 4 * half_step(rows) * 8 + 1e-4
    check_attention(gpu, workspace, rows, kind, 128, 16, 2, 64, counts, lengths, window=777)
    gpu.synchronize()


def test_attention_many_heads_of_one(gpu, workspace):
    check_attention(gpu, workspace, "bf16", "bf16", 64, 256, 1, 16, [2], [40])
    check_attention(gpu, workspace, "f32", "f32", 64, 24, 24, 16, [2, 1], [40, 70])
    check_attention(gpu, workspace, "f32", "bf16", 64, 17, 1, 16, [1, 1], [40, 170])


def test_attention_pool_past_32_bits(gpu, workspace):
    """Pages whose offsets take more than 32 bits, in elements."""
    pages, stride = 40, 1 << 27
    store = [torch.empty(pages * stride, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    pool = Pool(4, [550, 33], 16, 2, 64, "bf16", spare=0)
    pool.table[pool.table >= 0] = pages - 1 - pool.table[pool.table >= 0]
    big = [t.as_strided((pages, 16, 2, 64), (stride, 128, 64, 1)) for t in store]
    for t, i in zip(big, (1, 2)):
        t.copy_(normal(i, pages, 16, 2, 64, kind="bf16"))
    pool.keys, pool.values = big
    q = normal(3, 9, 4, 64, kind="bf16")
    for counts in ([8, 1], [1, 1]):
        n = sum(counts)
        batch = pool.batch(gpu, counts)
        out = torch.empty_like(q[:n])
        hip.paged_attention(gpu, pool.cache(gpu), batch, q[:n], out, workspace)
        want, bound, _ = attention(q[:n], pool.keys, pool.values, pool.offsets, pool.lengths, pool.table, 16, 1 / 8, 0,
                                   "bf16")
        within(out, want, bound)
    k = normal(5, 1, 2, 64, kind="bf16")
    one = hip.PagedBatch(gpu, ints([0, 1]), ints([1]), ints([[39]]), 1, 1, 1)
    hip.paged_append(gpu, pool.cache(gpu), one, k, k)
    assert torch.equal(pool.keys[39, 0], k[0]) and torch.equal(pool.values[39, 0], k[0])


def test_attention_refusals(gpu, workspace):
    pool = Pool(1, [20], 16, 2, 64, "bf16")
    cache, batch = pool.cache(gpu), pool.batch(gpu, [2])
    q = normal(1, 2, 4, 64, kind="bf16")
    out = torch.empty_like(q)

    def refused(call, message):
        with pytest.raises(hip.HipError, match=message) as info:
            call()
        assert info.value.status == hip.INVALID_ARGUMENT

    attend = hip.paged_attention
    refused(lambda: attend(gpu, cache, batch, q.half(), out.half(), workspace), "f32 rows read")
    refused(lambda: attend(gpu, cache, batch, q, out.half(), workspace), "outputs")
    refused(lambda: attend(gpu, cache, batch, q[:, :3], out[:, :3], workspace), "query heads")
    refused(lambda: attend(gpu, cache, batch, q, q, workspace), "overlap")
    refused(lambda: attend(gpu, cache, batch, q, out, workspace, gate=out), "overlap")
    refused(lambda: attend(gpu, cache, batch, q, out, workspace, scale=-1.0), "scale")
    refused(lambda: attend(gpu, cache, batch, q, out, workspace, scale=math.inf), "scale")
    refused(lambda: attend(gpu, cache, batch, q[:1], out[:1], workspace), "rows of shape")
    refused(lambda: attend(gpu, cache, batch, q[..., :32], out[..., :32], workspace), "rows of shape")
    refused(lambda: attend(gpu, cache, batch, q, out, workspace, gate=q.float()), "gate")
    wide = normal(1, 2, 4, 72, kind="bf16")
    refused(lambda: attend(gpu, cache, batch, wide[..., 4:68], out, workspace), "aligned")
    refused(lambda: attend(gpu, cache, batch, q.cpu(), out, workspace), "rows on cpu")
    closed = hip.PagedWorkspace(gpu, 1 << 20)
    closed.close()
    refused(lambda: attend(gpu, cache, batch, q, out, closed), "null")
    refused(lambda: hip.PagedWorkspace(gpu, 1000), "1 MiB")
    refused(lambda: hip.PagedCache(gpu, pool.keys, pool.values[:1]), "one type and layout")
    refused(lambda: hip.PagedCache(gpu, pool.keys.cpu(), pool.values.cpu()), "on cpu")
    refused(lambda: hip.PagedBatch(gpu, ints([0, 1]), ints([1, 2]), ints([[0], [1]]), 2, 1, 2), "offsets")
    refused(lambda: hip.PagedBatch(gpu, ints([0, 1]).long(), ints([1]), ints([[0]]), 1, 1, 1), "offsets")
    short = hip.PagedBatch(gpu, ints([0, 2]), ints([20]), ints([[0]]), 2, 2, 20)
    refused(lambda: attend(gpu, cache, short, q, out, workspace), "page table")
    odd = normal(1, 2, 24, 2, 64, kind="bf16")
    refused(lambda: attend(gpu, hip.PagedCache(gpu, odd, odd.clone()), batch, q, out, workspace), "page size")
    k = normal(1, 2, 2, 64, kind="bf16")
    append = hip.paged_append
    refused(lambda: append(gpu, cache, batch, k.half(), k.half()), "f32 rows go")
    refused(lambda: append(gpu, cache, batch, k, k.half()), "values")
    refused(lambda: append(gpu, cache, batch, k[:, :1], k), "rows of shape")
    refused(lambda: append(gpu, cache, batch, k, k, rope=hip.Rope(gpu, 128)), "more dimensions")
    refused(lambda: append(gpu, cache, batch, k, k, key_norm=torch.ones(64, device="cuda")), "norm weight")
    refused(lambda: append(gpu, cache, batch, k, k, epsilon=-1.0), "epsilon")
    refused(lambda: append(gpu, cache, batch, k, k, queries=q, queries_out=q.as_strided((2, 4, 64), (64, 128, 1))),
            "overlap")
    # nothing to do: no launch, no pointers needed
    none = hip.PagedBatch(gpu, ints([0]), torch.empty(0, dtype=torch.int32, device="cuda"),
                          torch.empty((0, 1), dtype=torch.int32, device="cuda"), 0, 0, 0)
    attend(gpu, cache, none, q[:0], out[:0], workspace)
    append(gpu, cache, none, k[:0], k[:0])


# ---- together: append, then attend ---------------------------------------------------

@pytest.mark.parametrize("rows,kind", PAIRS)
def test_a_prompt_in_chunks_then_single_tokens(gpu, workspace, rows, kind):
    """Two sequences' tokens appended and attended in uneven steps, single
    tokens last, give what one pass over all of them gives."""
    size, heads, kv, page, total = 128, 8, 2, 16, [75, 41]
    q, k, v = (normal(70 + i, sum(total), h, size, kind=rows) for i, h in enumerate((heads, kv, kv)))
    weight = normal(80, size, kind="bf16", scale=0.1)
    rope = hip.Rope(gpu, 64, "halves", 1e4)
    starts = [0, total[0]]
    pools = [Pool(90, total, page, kv, size, kind) for _ in range(2)]
    results = []
    for pool, steps in zip(pools, ([[75, 41]], [[30, 1], [1, 20], [41, 17], [1, 1], [1, 1], [1, 1]])):
        done, out = [0, 0], torch.empty_like(q)
        for counts in steps:
            at = np.concatenate([np.arange(starts[s] + done[s], starts[s] + done[s] + counts[s]) for s in range(2)])
            at = torch.tensor(at, device="cuda")
            done = [d + c for d, c in zip(done, counts)]
            batch = hip.PagedBatch(gpu, ints([0, counts[0], sum(counts)]), ints(done), ints(pool.table), sum(counts),
                                   max(counts), 80)
            rotated, o = torch.empty_like(q[at]), torch.empty_like(q[at])
            hip.paged_append(gpu, pool.cache(gpu), batch, k[at], v[at], rope, weight, q[at], weight, rotated)
            hip.paged_attention(gpu, pool.cache(gpu), batch, rotated, o, workspace)
            out[at] = o
        assert done == total
        results.append(out)
    for s in range(2):
        for p in range(total[s]):
            page_at = int(pools[0].table[s, p // page]), p % page
            assert torch.equal(pools[0].keys[page_at], pools[1].keys[page_at])
    offsets = np.array([0, total[0], sum(total)])
    position = torch.cat([torch.arange(n, device="cuda") for n in total])
    f, m = hip.rope_frequencies(64)
    rotated = turned(normalized(q, weight, 1.0, 1e-6), position, f, m, "halves")[0].to(TYPES[rows])
    want, bound, _ = attention(rotated, pools[0].keys, pools[0].values, offsets, total, pools[0].table, page,
                               1 / math.sqrt(size), 0, rows)
    # the queries' own roundings on the way (two half steps of their type, or
    # those of norm and rotation) move a score by as much of its sum of magnitudes
    moved = (2 * half_step(rows) if rows != "f32" else 32 * U) * 4.0 * math.sqrt(size) * 8
    for out in results:
        within(out, want, bound + 2 * math.expm1(2 * moved) * 4.0)


@pytest.mark.parametrize("rows,kind", [("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("chunk", [1, 24])
def test_captured_calls_replay_with_new_lengths(gpu, workspace, rows, kind, chunk):
    """Append and attention captured once and replayed while the lengths
    grow on the device, with eager work between: every replay equals the eager
    calls, also where a length has grown past the captured bound (NaN: 404 of
    400 entries in the last step of 24 tokens)."""
    size, heads, kv, page, top = 128, 8, 2, 16, 400
    table = ints(np.random.default_rng(1).permutation(60)[:50].reshape(2, 25))
    rope = hip.Rope(gpu, 128, "pairs", 1e4)
    stores = [[normal(i, 60, page, kv, size, kind=kind) for i in (1, 2)] for _ in range(2)]
    caches = [hip.PagedCache(gpu, *s) for s in stores]
    q, k, v = (normal(9, 2 * chunk, h, size, kind=rows) for h in (heads, kv, kv))
    lengths = ints([chunk, chunk + 9])
    batch = hip.PagedBatch(gpu, ints([0, chunk, 2 * chunk]), lengths, table, 2 * chunk, chunk, top)
    rotated, out = torch.empty_like(q), torch.empty_like(q)

    def step(cache, rotated, out, workspace):
        hip.paged_append(gpu, cache, batch, k, v, rope, queries=q, queries_out=rotated)
        hip.paged_attention(gpu, cache, batch, rotated, out, workspace)

    own = hip.PagedWorkspace(gpu, 8 << 20)
    step(caches[0], rotated, out, own)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            gpu.use_stream(torch.cuda.current_stream())
            step(caches[0], rotated, out, own)
    finally:
        gpu.use_stream(torch.cuda.current_stream())
    for store in stores[1:]:
        for a, b in zip(store, stores[0]):
            a.copy_(b)
    other = torch.empty_like(q), torch.empty_like(q)
    for growth in (0, 1, 90, 30, 250):
        lengths += growth
        for x, s in ((q, 3), (k, 4), (v, 5)):
            x.copy_(normal(s + growth, *x.shape, kind=rows))
        torch.cuda.synchronize()
        graph.replay()
        step(caches[1], *other, workspace)
        torch.cuda.synchronize()
        over = bool((lengths > top).any())
        assert bool(torch.isnan(out).any()) == over and over == (chunk == 24 and growth == 250)
        for a, b in ((out, other[1]), (rotated, other[0])):
            assert torch.equal(torch.nan_to_num(a, 99.0), torch.nan_to_num(b, 99.0))
        for a, b in zip(*stores):
            assert torch.equal(a, b)


def test_two_contexts_on_two_streams(gpu, workspace):
    """Calls of two contexts that run at once, each with its workspace, give
    what they give alone."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    pools = [Pool(40 + i, [4000, 3000], 32, 2, 128, "bf16") for i in range(2)]
    q = [normal(50 + i, 2, 16, 128, kind="bf16") for i in range(2)]
    want = []
    for pool, x in zip(pools, q):
        out = torch.empty_like(x)
        hip.paged_attention(gpu, pool.cache(gpu), pool.batch(gpu, [1, 1]), x, out, workspace)
        want.append(out)
    contexts = [hip.Context(0) for _ in range(2)]
    spaces = [hip.PagedWorkspace(c) for c in contexts]
    for c, s in zip(contexts, streams):
        c.use_stream(s)
    outs = [[torch.zeros_like(x) for _ in range(8)] for x in q]
    caches = [p.cache(c) for p, c in zip(pools, contexts)]
    batches = [p.batch(c, [1, 1]) for p, c in zip(pools, contexts)]
    torch.cuda.synchronize()
    for i in range(8):
        for j in range(2):
            hip.paged_attention(contexts[j], caches[j], batches[j], q[j], outs[j][i], spaces[j])
    for c in contexts:
        c.synchronize()
    for j in range(2):
        for o in outs[j]:
            assert torch.equal(o, want[j])
    for w, c in zip(spaces, contexts):
        w.close()
        c.close()


# ---- the full-attention layer over pages -----------------------------------------------

@pytest.fixture(scope="module")
def layer(gpu):
    from adi_amd import synthetic as syn
    rng = syn.rng_for(40, 256)
    tlut = syn.ne_tlut(rng)
    host = syn.full_attention(rng, 256, tlut)
    return host, hip.upload_full_attention(gpu, host, gpu.ne_codebook(tlut))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_layer_over_pages_is_the_layer_over_contiguous_caches(gpu, workspace, layer, kind):
    """Three sequences' prompts in chunks and single tokens in shared batches
    against full_attention_prefill of each over a contiguous cache. f32: the
    same caches to the roundings of an RMS norm's sums in another order, and
    outputs to 1e-4 of the largest (the layer tests' own bound). bf16: keys and
    values are off by half a step each, 2^-9 of themselves, which scores, weights
    and sums carry on linearly: 2^-5 of the largest output."""
    from adi_amd import synthetic as syn
    host, device = layer
    total, hidden, page = [90, 33, 7], host.hidden, 16
    x = [torch.from_numpy(syn.rms_normalized(syn.hidden_states(syn.rng_for(41, s), n, hidden))).cuda()
         for s, n in enumerate(total)]
    want, caches = [], []
    for rows in x:
        n = rows.shape[0]
        k = torch.zeros(n, 2, 256, device="cuda")
        v, out = torch.zeros_like(k), torch.empty(n, hidden, device="cuda")
        hip.full_attention_prefill(gpu, device, 0, n, rows, out, k, v, n)
        want.append(out)
        caches.append((k, v))
    pool = Pool(3, total, page, 2, 256, kind)
    done, got = [0, 0, 0], [torch.empty_like(w) for w in want]
    for counts in ([40, 0, 7], [1, 30, 0], [48, 1, 0], [1, 1, 0], [0, 1, 0]):
        rows = torch.cat([x[s][done[s]:done[s] + counts[s]] for s in range(3)])
        done = [d + c for d, c in zip(done, counts)]
        batch = hip.PagedBatch(gpu, ints(np.concatenate([[0], np.cumsum(counts)])), ints(done), ints(pool.table),
                               sum(counts), max(counts), 96)
        out = torch.empty(sum(counts), hidden, device="cuda")
        hip.full_attention_paged(gpu, device, pool.cache(gpu), batch, rows, out, workspace)
        at = 0
        for s in range(3):
            got[s][done[s] - counts[s]:done[s]] = out[at:at + counts[s]]
            at += counts[s]
    assert done == total
    limit = 1e-4 if kind == "f32" else 2.0 ** -5
    step = 64 * U if kind == "f32" else half_step("bf16") + 64 * U
    for s in range(3):
        scale = want[s].abs().amax(-1, keepdim=True)
        assert float(((got[s] - want[s]).abs() / scale).max()) <= limit, s
        for p in range(total[s]):
            at = int(pool.table[s, p // page]), p % page
            for mine, theirs in ((pool.keys[at], caches[s][0][p]), (pool.values[at], caches[s][1][p])):
                # turned pairs: relative to the pair, so to the head's largest
                assert float(((mine.float() - theirs).abs() / theirs.abs().amax(-1, keepdim=True)).max()) <= step


def test_layer_over_pages_refusals(gpu, workspace, layer):
    _, device = layer
    x = torch.zeros(2, 256, device="cuda")
    out = torch.empty_like(x)
    table = ints([[0, 1]])

    def call(pool, rows=x, to=out, tokens=2):
        cache = hip.PagedCache(gpu, pool, pool.clone())
        batch = hip.PagedBatch(gpu, ints([0, tokens]), ints([tokens]), table, tokens, tokens, 32)
        hip.full_attention_paged(gpu, device, cache, batch, rows, to, workspace)

    call(normal(1, 2, 16, 2, 256))
    for pool in (normal(1, 2, 16, 4, 256), normal(1, 2, 16, 2, 128), normal(1, 2, 16, 2, 256, kind="f16")):
        with pytest.raises(hip.HipError, match="2 heads of 256") as info:
            call(pool)
        assert info.value.status == hip.INVALID_ARGUMENT
    for rows, to in ((x[:1], out), (x.half(), out), (x, out.cpu()), (x, out.t())):
        with pytest.raises(hip.HipError, match="rows must be contiguous f32"):
            call(normal(1, 2, 16, 2, 256), rows, to)
    gpu.synchronize()


# ---- calls at the edges of what is allowed ------------------------------------------

@pytest.mark.parametrize("rows,kind", PAIRS)
def test_attention_of_more_sequences_than_lanes(gpu, workspace, rows, kind):
    """Chunks behind the 64th and the 128th sequence, beside single tokens
    and sequences without rows: a block finds its rows, a row its sequence."""
    counts = [1] * 70 + [0] * 5 + [9, 1, 0, 21] + [1] * 60 + [5]
    lengths = [7 + (11 * s) % 90 for s in range(len(counts))]
    lengths[-1] = 400
    check_attention(gpu, workspace, rows, kind, 64, 8, 2, 8, counts, lengths, padding=2)


@pytest.mark.parametrize("heads", [4, 64])
def test_a_bound_of_no_new_tokens(gpu, workspace, heads):
    """max_tokens 0: any sequence with rows is over it, so NaN, and appended nowhere."""
    pool = Pool(3, [20, 30], 16, 2, 64, "bf16", junk=None)
    before = pool.keys.clone()
    batch = hip.PagedBatch(gpu, ints([0, 3, 3]), ints([20, 30]), ints(pool.table), 4, 0, 32)
    q, k = normal(1, 4, heads, 64, kind="bf16"), normal(2, 4, 2, 64, kind="bf16")
    out = torch.full_like(q, 7.0)
    hip.paged_append(gpu, pool.cache(gpu), batch, k, k)
    hip.paged_attention(gpu, pool.cache(gpu), batch, q, out, workspace)
    assert torch.equal(pool.keys, before)
    assert bool(torch.isnan(out[:3]).all()) and bool((out[3:] == 7.0).all())


@pytest.mark.parametrize("heads,counts", [(4, [2, 1]), (32, [2, 40])])
def test_rows_before_the_first_sequence_stay(gpu, workspace, heads, counts):
    """offsets[0] above 0: the rows before it belong to no sequence either."""
    pool = Pool(4, [50, 90], 16, 2, 128, "f32", junk=None)
    n = sum(counts)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    q, k, v = normal(1, n + 3, heads, 128), normal(2, n + 3, 2, 128), normal(3, n + 3, 2, 128)
    out = []
    for shift in (0, 3):
        keys, values = pool.keys.clone(), pool.values.clone()
        cache = hip.PagedCache(gpu, keys, values)
        batch = hip.PagedBatch(gpu, ints(offsets + shift), ints([50, 90]), ints(pool.table), n + 3, max(counts), 96)
        rows = [torch.roll(x, shift, 0) for x in (q, k, v)]
        turned_rows, attended = torch.full_like(q, 5.0), torch.full_like(q, 7.0)
        hip.paged_append(gpu, cache, batch, rows[1], rows[2], queries=rows[0], queries_out=turned_rows)
        hip.paged_attention(gpu, cache, batch, rows[0], attended, workspace)
        out.append((keys, values, turned_rows[shift:shift + n], attended[shift:shift + n]))
        others = torch.cat([turned_rows[:shift] - 5, turned_rows[shift + n:] - 5, attended[:shift] - 7,
                            attended[shift + n:] - 7])
        assert bool((others == 0).all())
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 30, 1]])
def test_sequences_that_share_pages(gpu, workspace, rows, kind, counts):
    """One prefix's pages in several tables, and one page twice in a table:
    each row as if its sequence had copies of them."""
    lengths, page = [70, 100, 75], 16
    pool = Pool(6, lengths, page, 2, 64, kind, junk=None)
    apart = pool.keys.clone(), pool.values.clone()
    shared = pool.table.copy()
    shared[1, :3] = shared[2, :3] = shared[0, :3]
    shared[1, 3] = shared[1, 2]
    for s in range(3):
        for p in range(4):
            for x in apart:
                x[int(pool.table[s, p])] = x[int(shared[s, p])] if s else x[int(pool.table[s, p])]
    n = sum(counts)
    q = normal(7, n, 8, 64, kind=rows)
    out = torch.empty_like(q), torch.empty_like(q)
    pool.batch(gpu, counts)
    for table, (keys, values), to in ((shared, (pool.keys, pool.values), out[0]), (pool.table, apart, out[1])):
        batch = hip.PagedBatch(gpu, ints(np.concatenate([[0], np.cumsum(counts)])), ints(lengths), ints(table), n,
                               max(counts), 112)
        hip.paged_attention(gpu, hip.PagedCache(gpu, keys, values), batch, q, to, workspace)
    assert torch.equal(*out)


def test_attention_scale_refusals(gpu, workspace):
    pool = Pool(1, [20], 16, 2, 64, "bf16", junk=None)
    q = normal(1, 1, 4, 64, kind="bf16")
    batch = pool.batch(gpu, [1])
    for scale in (3e38, math.nan, -math.inf):
        with pytest.raises(hip.HipError, match="scale"):
            hip.paged_attention(gpu, pool.cache(gpu), batch, q, torch.empty_like(q), workspace, scale=scale)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("power", [12, 15, 20])
@pytest.mark.parametrize("counts", [[1], [40]])
def test_many_small_weights_add_up(gpu, workspace, rows, kind, power, counts):
    """One entry of weight 1 and thousands of 2^-power, f16's subnormal
    values among them (each exact in every type): none is lost, neither from the
    sums nor from the denominator."""
    def bend(pool, q):
        pool.keys.zero_()
        pool.values.fill_(1)
        first = int(pool.table[0, 0])
        pool.keys[first, 0, :, 0] = power
        pool.values[first, 0] = 0
        q.zero_()
        q[..., 0] = 1

    check_attention(gpu, workspace, rows, kind, 64, 4, 1, 64, counts, [6000], scale=math.log(2.0), bend=bend)
    # (a group of 64: more than a step's rows)
    check_attention(gpu, workspace, rows, kind, 128, 64, 1, 64, counts, [6000], scale=math.log(2.0), bend=bend)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("heads", [4, 64])
def test_weights_below_a_type_add_up_over_a_long_history(gpu, workspace, rows, kind, heads):
    """130,000 weights of 2^-26, half of f16's least value: their sum is as near
    as any other weights' are."""
    def bend(pool, q):
        pool.keys.zero_()
        pool.values.fill_(1)
        first = int(pool.table[0, 0])
        pool.keys[first, 0, :, 0] = 26
        pool.values[first, 0] = 0
        q.zero_()
        q[..., 0] = 1

    check_attention(gpu, workspace, rows, kind, 64, heads, 1, 64, [1], [130000], scale=math.log(2.0), bend=bend)


def test_layer_over_pages_keeps_bad_rows_to_themselves(gpu, workspace, layer):
    """A sequence over the batch's bounds, one with a bad page, rows of no
    sequence: NaN (or nothing of use) there, the others' rows as without them."""
    _, device = layer
    x = normal(5, 30, 256)
    pool = Pool(2, [40, 60, 25, 33], 16, 2, 256, "f32", junk=None)

    def call(lengths, table, pages):
        out = torch.empty_like(x)
        batch = hip.PagedBatch(gpu, ints([0, 9, 10, 21, 27]), ints(lengths), ints(table), 30, 12, 64)
        hip.full_attention_paged(gpu, device, hip.PagedCache(gpu, *pages), batch, x, out, workspace)
        return out

    good = call(pool.lengths, pool.table, (pool.keys.clone(), pool.values.clone()))
    table = pool.table.copy()
    table[2, 0] = 1 << 20
    bad = call([40, 65, 25, 33], table, (pool.keys.clone(), pool.values.clone()))
    assert bool(torch.isnan(bad[9:21]).all()) and bool(torch.isfinite(good[:27]).all())
    for rows in (slice(0, 9), slice(21, 27)):
        assert torch.equal(bad[rows], good[rows])


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("window", [0, 300])
def test_attention_of_steps_of_very_different_lengths(gpu, workspace, rows, kind, window):
    """Blocks shared by the lengths on the device: one long history among short
    and empty ones (whose one part each leaves few of the blocks), and
    all about alike."""
    for lengths in ([1 + s % 40 for s in range(29)] + [6000] + [0, 9, 0] + [5] * 26,
                    [900 + 31 * s for s in range(24)], [4000, 3], [2] * 64):
        counts = [1] * len(lengths)
        check_attention(gpu, workspace, rows, kind, 64, 8, 8, 16, counts, lengths, window=window)
    check_attention(gpu, workspace, rows, kind, 256, 4, 1, 64, [2, 0, 1, 3], [700, 50, 3000, 2], window=window)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("size", [64, 256])
def test_attention_of_both_kernels_in_one_call(gpu, workspace, rows, kind, size):
    """More single tokens than have room beside a chunk's blocks: those of
    large heads take the other kernel, of small ones a second round of the chunk's;
    with pages, windows and rows of no sequence as ever."""
    counts = [1] * 30 + [0, 40] + [1] * 30 + [2]
    lengths = [3 + (17 * s) % 150 for s in range(len(counts))]
    lengths[31], lengths[40], lengths[41] = 700, 1500, 0
    for window in (0, 60):
        gpu.profiling(True)
        check_attention(gpu, workspace, rows, kind, size, 32, 16, 16, counts, lengths, window=window, padding=3)
        ran = gpu.profile()
        gpu.profiling(False)
        assert "paged_chunk" in ran and ("paged_step" in ran or size == 64)


def test_captured_layer_replays_with_new_lengths(gpu, workspace, layer):
    """The layer over pages captured after a warm-up call, its replays against
    eager calls on a copy of the pool while the lengths grow."""
    _, device = layer
    stores = [[normal(i, 24, 16, 2, 256) for i in (1, 2)] for _ in range(2)]
    caches = [hip.PagedCache(gpu, *s) for s in stores]
    lengths, x = ints([5, 20, 9]), normal(3, 3, 256)
    table = ints(np.random.default_rng(2).permutation(24).reshape(3, 8))
    batch = hip.PagedBatch(gpu, ints([0, 1, 2, 3]), lengths, table, 3, 1, 128)
    out, want = torch.empty_like(x), torch.empty_like(x)
    own = hip.PagedWorkspace(gpu, 8 << 20)
    hip.full_attention_paged(gpu, device, caches[0], batch, x, out, own)
    hip.full_attention_paged(gpu, device, caches[1], batch, x, want, workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            gpu.use_stream(torch.cuda.current_stream())
            hip.full_attention_paged(gpu, device, caches[0], batch, x, out, own)
    finally:
        gpu.use_stream(torch.cuda.current_stream())
    for growth in (1, 1, 40, 60):
        lengths += growth
        x.copy_(normal(10 + growth, 3, 256))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        hip.full_attention_paged(gpu, device, caches[1], batch, x, want, workspace)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool(torch.isfinite(out).all())
        assert all(torch.equal(a, b) for a, b in zip(*stores))
